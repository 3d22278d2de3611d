// kv4.cuh -- kernels of a language-model layer between its projections at decode time: the
// per-head RMS norm and position rotation of queries and keys, the paged 4-bit key/value cache,
// and attention over that cache.
//
// Cache format.  A token's key (and value) of one kv head is cut into groups of 64 channels.  A
// group holds m = fp16(min x), s = fp16((max x - min x) / 15) and codes
// c = clamp(rint((x - m) / s), 0, 15); it stands for the values m + s c.  The codes of 16 tokens
// lie together in one tile, tiles of a (page, kv head) follow one another:
//   tile = K codes [16][hd / 2 bytes] | V codes [hd / 64][4][8][16 bytes] | scales [16][K s.., K m.., V s.., V m..] fp16
// A K row's 32-bit word holds 8 consecutive channels 64 gi + 8 r + j (nibble j, r = 0..7) and stands
// at byte (r / 2) * hd / 8 + (2 gi + r % 2) * 4, so that lane t of a quad finds the words of its
// 16-channel pieces side by side.  V is held the way the products over tokens take it: piece (t, r)
// of 16 bytes holds channels 64 gi + 8 r .. + 7 of tokens 2 t, 2 t + 8, 2 t + 1 and 2 t + 9, byte
// 4 i + b the two channels 2 i and 2 i + 1 of the b-th of these tokens.  A byte belongs to one
// token, so that appending never reads what is there.  The piece stands at t * 128 + (r ^ 2 t) * 16:
// a token's bytes share one line of 128, and a quarter warp's pieces (two r, four t) all banks.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "mma16.cuh"
#include "ptx.cuh"

namespace envg {

constexpr int KV_GROUP = 64;   // channels that share one scale and minimum
constexpr int KV_TILE = 16;    // tokens of a tile
constexpr float KV_HALF_MAX = 65504.0f;
// status[1] of an argument that only the device could see to be out of range
constexpr int SITE_KV_PAGE = 1001, SITE_KV_LEN = 1002, SITE_ROPE_POS = 1003;
constexpr int STATUS_ARG = -1;  // ENVG_ERR_ARG

__host__ __device__ constexpr int kv_tile_bytes(int hd) { return KV_TILE * (hd + 8 * (hd / KV_GROUP)); }

ENVG_DEV void kv_flag(int* status, int site) {
  if (status) {
    atomicExch(status, STATUS_ARG);
    atomicExch(status + 1, site);
  }
}

// The cache as the kernels see it, with the page table of one call.
struct Kv4View {
  uint8_t* base;
  int64_t pages;
  int page_size, kv_heads;
  FastDiv page_tiles;       // by the tiles of a page
  const int32_t* table;     // [batch][table_stride] page ids
  int64_t table_stride;
  const int32_t* ctx_lens;  // [batch] tokens held, this call's q_len new ones among them
  int* status;
};

// Tokens of sequence b; none where the length is not one that its row of the table can name, so that
// a wrong length cannot overwrite tokens that are held.
ENVG_DEV int kv_len(const Kv4View& c, int b) {
  const int n = __ldg(c.ctx_lens + b);
  if (n < 0 || n > c.table_stride * c.page_size) {
    kv_flag(c.status, SITE_KV_LEN);
    return 0;
  }
  return n;
}

// Tile of token `pos` of sequence b and kv head h; nullptr where the table names no page.
ENVG_DEV uint8_t* kv_tile(const Kv4View& c, int b, int h, int pos, int tile_bytes) {
  const uint32_t tile = (uint32_t)pos / KV_TILE, at = c.page_tiles.div(tile);
  const int32_t page = __ldg(c.table + (int64_t)b * c.table_stride + at);
  if (page < 0 || page >= c.pages) {
    kv_flag(c.status, SITE_KV_PAGE);
    return nullptr;
  }
  const int per_page = (int)c.page_tiles.d;
  return c.base + (((int64_t)page * c.kv_heads + h) * per_page + (int)(tile - at * per_page)) * tile_bytes;
}

// ---- norm of queries and keys per head + position rotation ------------------------------------
// y = rot(x w / sqrt(mean x^2 + eps)); rot turns the pair (a, b) of channels into
// (a cos - b sin, b cos + a sin).  A pair is (i, i + hd/2), or (2i, 2i + 1) when interleaved.
// A thread holds eight channels (four pairs) of NR_HEADS heads of one token: a head's pairs never
// leave their thread, the norm is one shuffle tree over hd / 8 threads (rounded up to a power of
// two), and weights and angles are read once for the heads.  HBM bounds it: every load is issued
// before the first use (4608 x 48 heads of 128: 40.8 us, 5.6 TB/s; with one head to a thread it was
// bound by instructions and by L1, at 51 us).
constexpr int NR_HEADS = 4;
struct NormRopeArgs {
  float *qd, *kd;
  const float *q, *k;
  int64_t ldqd, ldkd, ldq, ldk;
  const float *wq, *wk, *cos, *sin;
  int64_t table_rows;
  const int32_t* positions;
  int64_t pos0, tokens;
  int heads, kv_heads, hd;
  float eps, by_hd;  // by_hd: 1 / hd
  int interleaved, vec;
  int q_runs;         // runs of NR_HEADS heads of q; k's follow
  FastDiv per_token;  // by the runs of a token
  int* status;
};

template <int LANES>
__global__ void __launch_bounds__(256) k_qk_norm_rope(const NormRopeArgs a) {
  griddep_wait();
  griddep_launch_dependents();
  const uint32_t item = (blockIdx.x * 256u + threadIdx.x) / LANES;  // (token, run of heads)
  const int li = threadIdx.x % LANES;
  const uint32_t tk = a.per_token.div(item);
  const int64_t tok = tk;
  const int run = (int)(item - tk * a.per_token.d);
  const bool isq = run < a.q_runs, vec = a.vec != 0;
  const int h0 = (isq ? run : run - a.q_runs) * NR_HEADS, left = (isq ? a.heads : a.kv_heads) - h0;
  const int n = tok < a.tokens && 8 * li < a.hd ? min(left, NR_HEADS) : 0;  // heads of this thread
  // channels 4 li .. + 3 and hd / 2 + 4 li .. + 3: four pairs (i, i + hd / 2), or two and two pairs
  // (2 i, 2 i + 1) when interleaved
  const int i0 = 4 * li, i1 = a.hd / 2 + 4 * li;
  const float* src = isq ? a.q + tok * a.ldq : a.k + tok * a.ldk;
  float4 x0[NR_HEADS], x1[NR_HEADS];
#pragma unroll
  for (int j = 0; j < NR_HEADS; ++j) {
    x0[j] = x1[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (j < n) x0[j] = ld_f4(src + (int64_t)(h0 + j) * a.hd + i0, vec), x1[j] = ld_f4(src + (int64_t)(h0 + j) * a.hd + i1, vec);
  }
  float4 w0 = make_float4(1.f, 1.f, 1.f, 1.f), w1 = w0, c = w0, s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (n > 0) {
    const float* w = isq ? a.wq : a.wk;
    if (w) w0 = ld_f4(w + i0, vec), w1 = ld_f4(w + i1, vec);
    if (a.cos) {
      int64_t pos = a.positions ? (int64_t)__ldg(a.positions + tok) : a.pos0 + tok;
      if (pos < 0 || pos >= a.table_rows) {
        kv_flag(a.status, SITE_ROPE_POS);
        pos = pos < 0 ? 0 : a.table_rows - 1;
      }
      const float *cp = a.cos + pos * (a.hd / 2), *sp = a.sin + pos * (a.hd / 2);
      if (!a.interleaved) {
        c = ld_f4(cp + 4 * li, vec), s = ld_f4(sp + 4 * li, vec);
      } else {  // pairs 2 li, 2 li + 1 and hd / 4 + 2 li, + 1
        const int f0 = 2 * li, f1 = a.hd / 4 + 2 * li;
        c = make_float4(cp[f0], cp[f0 + 1], cp[f1], cp[f1 + 1]);
        s = make_float4(sp[f0], sp[f0 + 1], sp[f1], sp[f1 + 1]);
      }
    }
  }
  float ss[NR_HEADS];
#pragma unroll
  for (int j = 0; j < NR_HEADS; ++j) {
    const float4 u = x0[j], v = x1[j];
    float q = u.x * u.x;
    q = fmaf(u.y, u.y, q), q = fmaf(u.z, u.z, q), q = fmaf(u.w, u.w, q);
    q = fmaf(v.x, v.x, q), q = fmaf(v.y, v.y, q), q = fmaf(v.z, v.z, q), q = fmaf(v.w, v.w, q);
    ss[j] = q;
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1)
#pragma unroll
    for (int j = 0; j < NR_HEADS; ++j) ss[j] += __shfl_xor_sync(0xffffffffu, ss[j], o);
  float* dst = isq ? a.qd + tok * a.ldqd : a.kd + tok * a.ldkd;
#pragma unroll
  for (int j = 0; j < NR_HEADS; ++j) {
    if (j >= n) break;
    const float inv = 1.0f / sqrtf(ss[j] * a.by_hd + a.eps);
    float4 u = x0[j], v = x1[j];
    u = make_float4(u.x * inv * w0.x, u.y * inv * w0.y, u.z * inv * w0.z, u.w * inv * w0.w);
    v = make_float4(v.x * inv * w1.x, v.y * inv * w1.y, v.z * inv * w1.z, v.w * inv * w1.w);
    if (a.cos) {
      if (a.interleaved) {
        u = make_float4(u.x * c.x - u.y * s.x, u.y * c.x + u.x * s.x, u.z * c.y - u.w * s.y, u.w * c.y + u.z * s.y);
        v = make_float4(v.x * c.z - v.y * s.z, v.y * c.z + v.x * s.z, v.z * c.w - v.w * s.w, v.w * c.w + v.z * s.w);
      } else {
        const float4 p = u;
        u = make_float4(p.x * c.x - v.x * s.x, p.y * c.y - v.y * s.y, p.z * c.z - v.z * s.z, p.w * c.w - v.w * s.w);
        v = make_float4(v.x * c.x + p.x * s.x, v.y * c.y + p.y * s.y, v.z * c.z + p.z * s.z, v.w * c.w + p.w * s.w);
      }
    }
    st_f4(dst + (int64_t)(h0 + j) * a.hd + i0, u, vec);
    st_f4(dst + (int64_t)(h0 + j) * a.hd + i1, v, vec);
  }
}

// ---- cache: write and read ----------------------------------------------------------------------
// Eight threads hold one group of 64 channels, eight consecutive channels (one word of codes)
// each; the group's minimum and maximum are one shuffle tree.  Codes are those of the IEEE quotient
// rounded to nearest even, so equal inputs give equal codes on any path that uses the formula; the
// quotient itself is taken only where a product with the reciprocal comes near a half.
ENVG_DEV uint32_t kv_k_word(int hd, int tok, int gi, int r) {
  return tok * (hd / 2) + (r >> 1) * (hd / 8) + (2 * gi + (r & 1)) * 4;
}
// First of the four bytes (4 apart) of V's channels 64 gi + 8 r .. + 7 of a token.
ENVG_DEV uint32_t kv_v_byte(int hd, int tok, int gi, int r) {
  const int t = (tok & 7) >> 1;
  return KV_TILE * (hd / 2) + gi * 512 + t * 128 + ((r ^ (2 * t)) * 16) + (tok >> 3) + 2 * (tok & 1);
}
// Byte offset of the scale of (token, K or V, group); its minimum stands hd / 64 halves further.
ENVG_DEV uint32_t kv_scale_at(int hd, int tok, int v, int gi) { return KV_TILE * hd + tok * (hd / 8) + v * (hd / 16) + 2 * gi; }

struct KvRowsArgs {
  Kv4View c;
  float *k, *v;  // [batch * q_len, ld], read by the append and written by the read
  int64_t ldk, ldv;
  int hd, batch, q_len, vec;
  int runs, runs_per;    // runs of ROWS new tokens in all, and of a block
  FastDiv per_run, seq;  // by a run's threads (eight for each K or V, head and group), by a sequence's runs
};

// A thread takes ROWS consecutive tokens, so that most find their tile where the last one's was
// (one token to a thread spent two thirds of its instructions on finding it).  4096 tokens, 8 heads
// of 128, written and read back: 23.9 us, 3.2 TB/s over both kernels, bound by instructions; 7.6 us
// more with V's bytes of a token in four lines instead of one.
template <bool READ, int ROWS>
__global__ void __launch_bounds__(256) k_kv4_rows(const KvRowsArgs a) {
  griddep_wait();
  griddep_launch_dependents();
  const int G = a.hd / KV_GROUP, lg = G - 1;
  // a block takes as many whole runs as it has threads for, or a part of one (blockIdx.y)
  const uint32_t in_block = blockIdx.y * 256u + threadIdx.x, rb = a.per_run.div(in_block);
  const int run0 = blockIdx.x * a.runs_per + (int)rb;
  const bool work = rb < (uint32_t)a.runs_per && run0 < a.runs;
  const uint32_t run = work ? run0 : 0;
  const int unit = work ? (int)(in_block - rb * a.per_run.d) / 8 : 0;
  const int r = threadIdx.x % 8;
  const int isv = unit >= a.c.kv_heads * G ? 1 : 0, n = unit - isv * a.c.kv_heads * G;
  const int gi = n & lg, h = n >> lg;
  const int b = (int)a.seq.div(run);
  const int i0 = (int)(run - (uint32_t)b * a.seq.d) * ROWS, rows = work ? min(ROWS, a.q_len - i0) : 0;
  const bool vec = a.vec != 0;
  const int64_t ld = isv ? a.ldv : a.ldk;
  float* at = (isv ? a.v : a.k) + ((int64_t)b * a.q_len + i0) * ld + (int64_t)h * a.hd + gi * KV_GROUP + 8 * r;
  float4 p0[ROWS], p1[ROWS];
  if (!READ) {  // under way while the page is looked up
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      p0[i] = p1[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i < rows) p0[i] = ld_f4(at + i * ld, vec), p1[i] = ld_f4(at + i * ld + 4, vec);
    }
  }
  const int pos0 = kv_len(a.c, b) - a.q_len + i0;
  const int tile_bytes = kv_tile_bytes(a.hd);
  uint8_t* tile = nullptr;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int pos = pos0 + i, tok = pos & (KV_TILE - 1);
    const bool on = i < rows && pos >= 0;
    if (on && (i == 0 || tok == 0 || pos == 0)) tile = kv_tile(a.c, b, h, pos, tile_bytes);
    uint8_t* codes = tile + (isv ? kv_v_byte(a.hd, tok, gi, r) : kv_k_word(a.hd, tok, gi, r));
    uint8_t* scale = tile + kv_scale_at(a.hd, tok, isv, gi);
    if (READ) {
      if (i >= rows) return;
      float x[8] = {};
      if (on && tile) {
        uint32_t w;
        if (isv) w = codes[0] | codes[4] << 8 | codes[8] << 16 | (uint32_t)codes[12] << 24;
        else w = *reinterpret_cast<const uint32_t*>(codes);
        const __half* sp = reinterpret_cast<const __half*>(scale);
        const float s = __half2float(sp[0]), m = __half2float(sp[G]);
#pragma unroll
        for (int j = 0; j < 8; ++j)  // a code in the low bits of 2^23
          x[j] = fmaf(s, __uint_as_float(and_or(w >> (4 * j), 15u, 0x4B000000u)) - 8388608.0f, m);
      }
      st_f4(at + i * ld, make_float4(x[0], x[1], x[2], x[3]), vec);
      st_f4(at + i * ld + 4, make_float4(x[4], x[5], x[6], x[7]), vec);
    } else {
      const float x[8] = {p0[i].x, p0[i].y, p0[i].z, p0[i].w, p1[i].x, p1[i].y, p1[i].z, p1[i].w};
      float lo = x[0], hi = x[0];
      bool nan = x[0] != x[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) lo = fminf(lo, x[j]), hi = fmaxf(hi, x[j]), nan |= x[j] != x[j];
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      }
      const uint32_t any = (__ballot_sync(0xffffffffu, nan) >> (threadIdx.x & 24)) & 0xffu;
      if (on && tile) {
        if (any) lo = hi = __int_as_float(0x7fc00000);  // a group with a NaN holds NaN
        const float low = lo < -KV_HALF_MAX ? -KV_HALF_MAX : lo > KV_HALF_MAX ? KV_HALF_MAX : lo;
        const float step = __fdiv_rn(__fsub_rn(hi, lo), 15.0f);
        const __half hs = __float2half_rn(step > KV_HALF_MAX ? KV_HALF_MAX : step), hm = __float2half_rn(low);
        const float s = __half2float(hs), m = __half2float(hm);
        uint32_t w = 0;
        if (s > 0.0f) {
          const float inv = __frcp_rn(s), whole = 12582912.0f;  // 1.5 x 2^23: adding it rounds to an integer
          bool near = false;
          uint32_t c[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float q = fminf(fmaxf(__fsub_rn(x[j], m) * inv, 0.0f), 15.0f), y = __fadd_rn(q, whole);
            c[j] = __float_as_uint(y);
            // the product is within 15 x 2^-22 of the quotient: near a half, divide
            near |= fabsf(__fsub_rn(q, __fsub_rn(y, whole))) > 0.5f - 1e-5f;
          }
          if (near)
#pragma unroll
            for (int j = 0; j < 8; ++j)
              c[j] = __float_as_uint(__fadd_rn(fminf(fmaxf(__fdiv_rn(__fsub_rn(x[j], m), s), 0.0f), 15.0f), whole));
#pragma unroll
          for (int j = 0; j < 8; ++j) w |= (c[j] & 15u) << (4 * j);
        }
        if (isv) {
#pragma unroll
          for (int j = 0; j < 4; ++j) codes[4 * j] = (uint8_t)(w >> (8 * j));
        } else {
          *reinterpret_cast<uint32_t*>(codes) = w;
        }
        if (r == 0) {
          __half* sp = reinterpret_cast<__half*>(scale);
          sp[0] = hs, sp[G] = hm;
        }
      }
    }
  }
}

// ---- attention over the cache ---------------------------------------------------------------
// Query token i of sequence b stands at p = ctx_lens[b] - q_len + i and sees the cached tokens
// j <= p, with a window W > 0 only those with j > p - W or j < sinks.  A row that sees nothing
// gives zeros.
struct KvAttnArgs {
  Kv4View c;
  const float* q;
  float* out;
  int64_t ldq, ldo;
  int batch, q_len, heads, hd, window, sinks;
  float sl2;  // softmax scale * log2 e
  int vec, vec_out;        // rows of q, of out are 16-byte aligned
  int splits, log_splits;  // CTAs of a cluster, a power of two: parts of the tokens
  uint64_t wait_cap_ns;
};

// k_kv4_attn: flash attention of up to 4 NB query rows over one kv head's cached tokens.
//
// Mathematics.  The rows are (query token, head) pairs that read the same kv head.  A row's score
// of token j is sum_g s_jg (q_g . c_jg) + m_jg sum(q_g) over its groups of 64 channels, and its
// output sum_j p_j (s_jg (c_jg - 8) + (m_jg + 8 s_jg)).  Both products with codes run on the
// tensor cores as 8-bit integer m16n8k32 products, whose 32-bit sums are exact.  The codes are the
// unsigned 16-row operand (16 tokens of K, 16 channels of V^T), four of them unpacked by one or two
// logic operations, once for all rows.  The other factor is the 8-column one, a fixed-point number
// cut into digits to the base 256: q with 31 bits of its group's largest value in four signed
// digits (two products of two adjacent columns a row), p s with 22 bits of its group's largest in the
// unit in three unsigned ones.  A thread joins its digits' sums, which are one row's, in integers and
// converts once.  The c - 8 of the output comes from a start of the sums at -8 sum(p s), itself a
// product (sums of the positive codes would be far larger than the result and cost its last bits).
// Scores come out as [token][row]; an 8 x 8 transpose in registers (movmatrix) makes the p s operand
// of them.
//
// Split.  Tokens are taken in units of two 16-token tiles, dealt out over the warps of a cluster
// of CTAs (one cluster per sequence, kv head and 4 NB rows).  Each warp runs a one-pass softmax
// with its own ring of bulk copies; the warps' (max, sum, output) are joined in shared memory, the
// CTAs' through distributed shared memory in rank order: no workspace, no atomics, one launch.
//
// Rounding.  Both fixed-point numbers are relative to the largest of one group of 64 channels, whose
// sums are the only ones they enter: q to 2^-30 of it, p s to 2^-22, where a step of V's own codes is
// a fifteenth of the group's span.  One unit for both groups of a 128-channel head lost log2 R bits in
// a group R times smaller.
//
// Bound: the chain of dependent steps of each warp (about 455 instructions a unit and warp for four
// rows; with four CTAs per SM, as many as registers allow, issue slots are 56% busy, DRAM 47%, the
// tensor pipe 26%), and start and join around it (6 us alone, a quarter of the instructions below).
// Measured: 16 sequences of 8192 to 16384 tokens, 32 / 8 heads of 128: 55 to 58 us, 4.1 TB/s; fp16
// operands with q and p s in two parts took 68 (9 operations to unpack 8 codes against 3).
constexpr int KVA_WARPS = 4, KVA_THREADS = 32 * KVA_WARPS, KVA_STAGES = 2;
constexpr int SITE_KVA_RING = 60;  // status[1] of a ring wait that ran out

template <int HD, int NB>
struct KvaSmem {
  static constexpr int ROWS = 4 * NB;
  static constexpr int TILE = kv_tile_bytes(HD), STAGE = 2 * TILE;
  static constexpr int RING = KVA_STAGES * STAGE;  // per warp
  // the rings are empty when the outputs of the warps are joined: [warp][ROWS][HD], then the CTA's
  static constexpr int OUT_LD = HD + 4, OUT = (KVA_WARPS + 1) * ROWS * OUT_LD * 4;
  static constexpr int BARS = KVA_WARPS * RING > OUT ? KVA_WARPS * RING : OUT;  // mbarriers
  static constexpr int ABORT = BARS + KVA_WARPS * KVA_STAGES * 8;               // abort flag of the bounded waits
  static constexpr int ML = ABORT + 16;                                         // [warps + 1][max ROWS | sum ROWS]
  static constexpr int TOTAL = ML + (KVA_WARPS + 1) * 2 * ROWS * 4;
};

template <int HD, int NB>
__global__ void __launch_bounds__(KVA_THREADS, NB == 1 ? 4 : 3) k_kv4_attn(const KvAttnArgs a) {
  using S = KvaSmem<HD, NB>;
  constexpr int G = HD / KV_GROUP;  // groups per head
  constexpr int ROWS = S::ROWS;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t sbase = smem_u32(smem);
  const uint32_t ring = sbase + warp * S::RING, bars = sbase + S::BARS + warp * KVA_STAGES * 8;
  volatile int* abort_s = reinterpret_cast<volatile int*>(smem + S::ABORT);
  float* ml = reinterpret_cast<float*>(smem + S::ML);
  if (lane == 0)
    for (int i = 0; i < KVA_STAGES; ++i) mbar_init(bars + 8 * i, 2);
  if (threadIdx.x == 0) *abort_s = 0;
  fence_mbar_init();
  griddep_wait();
  griddep_launch_dependents();
  __syncthreads();

  const int splits = a.splits, rank = blockIdx.x & (splits - 1), row_tile = blockIdx.x >> a.log_splits, b = blockIdx.y;
  const int per_kv = a.heads / a.c.kv_heads, rows = per_kv * a.q_len;
  const int kvh = row_tile % a.c.kv_heads, row0 = (row_tile / a.c.kv_heads) * ROWS;
  // q first: its loads are under way while the lengths and the page table are looked up
  float x[NB][16 * G];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int rr = row0 + 4 * nb + (g >> 1);
    const bool have = rr < rows;
    const int qi = have ? rr / per_kv : 0, qh = kvh * per_kv + (have ? rr - qi * per_kv : 0);
    const float* src = a.q + ((int64_t)b * a.q_len + qi) * a.ldq + (int64_t)qh * HD + 16 * t;
#pragma unroll
    for (int i = 0; i < 4 * G; ++i) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (have) v = ld_f4(src + 64 * (i / 4) + 4 * (i % 4), a.vec != 0);
      x[nb][4 * i] = v.x, x[nb][4 * i + 1] = v.y, x[nb][4 * i + 2] = v.z, x[nb][4 * i + 3] = v.w;
    }
  }
  const int len = kv_len(a.c, b);
  // tiles that some row of the CTA sees: the first n_sink ones, then [first, last]
  const int p_lo = len - a.q_len + row0 / per_kv, p_hi = len - a.q_len + min(rows - 1, row0 + ROWS - 1) / per_kv;
  const int lo = a.window > 0 ? max(0, p_lo - a.window + 1) : 0;
  const int first = lo / KV_TILE;
  const int n_sink = a.window > 0 ? min((a.sinks + KV_TILE - 1) / KV_TILE, first) : 0;
  const int n_tiles = p_hi < 0 ? 0 : n_sink + p_hi / KV_TILE - first + 1;
  const int units = (n_tiles + 1) / 2, stride = splits * KVA_WARPS, u0 = rank * KVA_WARPS + warp;

  // Ring of bulk copies.  Sixteen units at a time, each lane looks up one tile and later brings it:
  // lanes 2 (n % 16) and 2 (n % 16) + 1 those of the warp's n-th unit.
  const int per_page = a.c.page_size / KV_TILE;
  const int32_t* table = a.c.table + (int64_t)b * a.c.table_stride;
  const int mine = u0 < units ? (units - u0 + stride - 1) / stride : 0;  // units of this warp
  auto tile_at = [&](int batch) { const int i = 2 * (u0 + (16 * batch + (lane >> 1)) * stride) + (lane & 1); return i >= n_tiles ? -1 : i < n_sink ? i : first + i - n_sink; };
  auto look_up = [&](int batch) -> int32_t {
    const int tile = 16 * batch < mine ? tile_at(batch) : -1;
    return tile >= 0 ? __ldg(table + tile / per_page) : -1;
  };
  int32_t ahead = look_up(0);
  const uint8_t* src = nullptr;
  uint32_t there = 0, there_next = 0;  // tiles that exist: of the batch being worked on, being brought
  auto issue = [&](int n, int st) {
    if ((n & 15) == 0) {
      const int tile = tile_at(n >> 4);
      bool ok = tile >= 0;
      if (ok && (ahead < 0 || ahead >= a.c.pages)) {
        kv_flag(a.c.status, SITE_KV_PAGE);
        ok = false;
      }
      src = ok ? a.c.base + (((int64_t)ahead * a.c.kv_heads + kvh) * per_page + tile % per_page) * S::TILE : nullptr;
      there_next = __ballot_sync(0xffffffffu, ok);
      ahead = look_up((n >> 4) + 1);
    }
    if ((lane >> 1) == (n & 15)) {
      const uint32_t bar = bars + 8 * st;
      if (src) {
        mbar_arrive_expect_tx(bar, S::TILE);
        bulk_load(ring + st * S::STAGE + (lane & 1) * S::TILE, src, S::TILE, bar);
      } else {
        mbar_arrive(bar);
      }
    }
  };
  for (int n = 0; n < KVA_STAGES && n < mine; ++n) issue(n, n);
  // tiles [w_lo, w_hi) and [0, w_sink) of the list are seen whole by every row of the CTA
  const int w_hi = n_sink + (p_lo + 1) / KV_TILE - first, w_sink = min(n_sink, a.sinks / KV_TILE);
  const int w_lo = n_sink + (a.window > 0 ? max(0, p_hi - a.window) / KV_TILE + 1 - first : 0);

  // q: columns g of the two operands are digits g % 2 and 2 + g % 2 of row g / 2, in the order of
  // the K words' nibbles; a thread's scores are those of row t
  uint32_t qb[NB][2 * G][2][2];
  float qs[NB][G], cq[NB][G];
  int pos[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int from = 8 * t;  // a lane whose g / 2 is this thread's t
    float up[G];
#pragma unroll
    for (int gi = 0; gi < G; ++gi) {  // each group has a unit of its own, as its scores have a scale of their own
      uint32_t top = 0;
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 16; ++j) top = max(top, __float_as_uint(x[nb][16 * gi + j]) & 0x7fffffffu), sum += x[nb][16 * gi + j];
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o)), sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const int e = min(126, fixed_exp(__uint_as_float(top)));  // scores of a row below 2^-97 are zero to fp32
      up[gi] = pow2(e);
      qs[nb][gi] = __shfl_sync(0xffffffffu, sum, from) * a.sl2;
      // a row with an infinity or a NaN gives NaN
      cq[nb][gi] = __shfl_sync(0xffffffffu, top >= 0x7f800000u ? __int_as_float(0x7fc00000) : pow2(-e), from) * a.sl2;
    }
    const int mr = row0 + 4 * nb + t;
    pos[nb] = mr < rows ? len - a.q_len + mr / per_kv : -1;
    const uint32_t pick[2] = {(g & 1) ? 0x0051u : 0x0040u, (g & 1) ? 0x0073u : 0x0062u};
#pragma unroll
    for (int w = 0; w < 2 * G; ++w) {
      uint32_t d[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = digits256(__float2int_rn(x[nb][8 * w + j] * up[w / 2]));
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h)  // nibbles 0, 2, 4, 6 and 1, 3, 5, 7
          qb[nb][w][n][h] = __byte_perm(__byte_perm(d[h], d[2 + h], pick[n]), __byte_perm(d[4 + h], d[6 + h], pick[n]), 0x5410);
    }
  }

  // sums of a row are held relative to 2^m, m its largest score so far rounded up to a whole power
  float o[NB][4 * G][2], m[NB], l[NB], pm[NB][G];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    m[nb] = -INFINITY, l[nb] = 0.0f;
#pragma unroll
    for (int gi = 0; gi < G; ++gi) pm[nb][gi] = 0.0f;
#pragma unroll
    for (int i = 0; i < 4 * G; ++i) o[nb][i][0] = o[nb][i][1] = 0.0f;
  }
  const WaitCtl wc{a.wait_cap_ns, a.c.status, abort_s, 0};
  const uint32_t nib = in_register(0x0F0F0F0Fu);
  bool fine = true;
  int st = 0;
  uint32_t phase = 0;
  for (int n = 0; n < mine; ++n) {
    const int unit = u0 + n * stride;
    fine = wait_bounded(bars + 8 * st, phase, wc, SITE_KVA_RING);
    if (!__all_sync(0xffffffffu, fine)) {
      fine = false;
      break;
    }
    const uint8_t* stage = smem + warp * S::RING + st * S::STAGE;
    if ((n & 15) == 0) there = there_next;
    const uint32_t vote = (there >> (2 * (n & 15))) & 3u;
    // scores of tokens g and g + 8 of each tile, log2 units
    float x[NB][2][2], vs[2][2][G], vm[2][2][G];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      const uint8_t* tile = stage + tt * S::TILE;
      float ks[2][G], km[2][G];
      uint32_t kw[2][2 * G];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint8_t* p = tile + KV_TILE * HD + (g + 8 * i) * (HD / 8);
        const uint8_t* pk = tile + (g + 8 * i) * (HD / 2) + t * (HD / 8);
        if (G == 2) {
          const uint4 u = *reinterpret_cast<const uint4*>(p);
          const float2 f0 = __half22float2(bits_h2(u.x)), f1 = __half22float2(bits_h2(u.y));
          const float2 f2 = __half22float2(bits_h2(u.z)), f3 = __half22float2(bits_h2(u.w));
          ks[i][0] = f0.x, ks[i][G - 1] = f0.y, km[i][0] = f1.x, km[i][G - 1] = f1.y;
          vs[tt][i][0] = f2.x, vs[tt][i][G - 1] = f2.y, vm[tt][i][0] = f3.x, vm[tt][i][G - 1] = f3.y;
          const uint4 k4 = *reinterpret_cast<const uint4*>(pk);
          kw[i][0] = k4.x, kw[i][1] = k4.y, kw[i][2 * G - 2] = k4.z, kw[i][2 * G - 1] = k4.w;
        } else {
          const uint2 u = *reinterpret_cast<const uint2*>(p);
          const float2 f0 = __half22float2(bits_h2(u.x)), f1 = __half22float2(bits_h2(u.y));
          ks[i][0] = f0.x, km[i][0] = f0.y, vs[tt][i][0] = f1.x, vm[tt][i][0] = f1.y;
          const uint2 k2 = *reinterpret_cast<const uint2*>(pk);
          kw[i][0] = k2.x, kw[i][1] = k2.y;
        }
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          x[nb][tt][i] = qs[nb][0] * km[i][0];
          if (G == 2) x[nb][tt][i] = fmaf(qs[nb][G - 1], km[i][G - 1], x[nb][tt][i]);
        }
#pragma unroll
      for (int gi = 0; gi < G; ++gi) {
        int d[NB][2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int w = 2 * gi + h;
          const uint32_t a0 = kw[0][w] & nib, a1 = kw[1][w] & nib, a2 = (kw[0][w] >> 4) & nib, a3 = (kw[1][w] >> 4) & nib;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              if (h == 0) mma_u8s8<true>(d[nb][k], a0, a1, a2, a3, qb[nb][w][k][0], qb[nb][w][k][1]);
              else mma_u8s8<false>(d[nb][k], a0, a1, a2, a3, qb[nb][w][k][0], qb[nb][w][k][1]);
            }
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float dot = fmaf((float)(d[nb][1][2 * i + 1] * 256 + d[nb][1][2 * i]), 65536.0f, (float)(d[nb][0][2 * i + 1] * 256 + d[nb][0][2 * i]));
            x[nb][tt][i] = fmaf(dot * cq[nb][gi], ks[i][gi], x[nb][tt][i]);
          }
      }
    }
    // masks: only where a row of the CTA does not see the whole unit.  A row hides a token by its
    // score; its scale and minimum are dropped where no row sees it (they may hold anything there).
    const bool whole = vote == 3u && ((2 * unit >= w_lo && 2 * unit + 1 < w_hi) || 2 * unit + 1 < w_sink);
    if (!whole) {
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int at = 2 * unit + tt, j = (at < n_sink ? at : first + at - n_sink) * KV_TILE + g + 8 * i;
          bool any = false;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            const bool see = ((vote >> tt) & 1u) && j <= pos[nb] && (a.window <= 0 || j > pos[nb] - a.window || j < a.sinks);
            if (!see) x[nb][tt][i] = -INFINITY;
            any |= see;
          }
#pragma unroll
          for (int gi = 0; gi < G; ++gi)
            if (!any) vs[tt][i][gi] = vm[tt][i][gi] = 0.0f;
        }
    }
    float top[NB];
    bool moves = false;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      top[nb] = fmaxf(fmaxf(x[nb][0][0], x[nb][0][1]), fmaxf(x[nb][1][0], x[nb][1][1]));
      moves |= top[nb] > m[nb];
    }
    if (__any_sync(0xffffffffu, moves)) {  // a larger score: the sums so far are scaled down to it
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) top[nb] = fmaxf(top[nb], __shfl_xor_sync(0xffffffffu, top[nb], off));
        const float m2 = fmaxf(m[nb], ceilf(top[nb]));
        const float alpha = m[nb] == -INFINITY ? 0.0f : ex2(m[nb] - m2);
        m[nb] = m2;
        l[nb] *= alpha;
#pragma unroll
        for (int gi = 0; gi < G; ++gi) pm[nb][gi] *= alpha;
#pragma unroll
        for (int i = 0; i < 4 * G; ++i) o[nb][i][0] *= alpha, o[nb][i][1] *= alpha;
      }
    }
    uint32_t pb[NB][G][2][2];  // [operand][tile]
    float f[NB][G];            // what one unit of the weights' fixed-point numbers stands for
    // a token that one thread's row sees may be hidden from its other rows: 0 x NaN must not come
    // through there (with one row to a thread, what it does not see is zero already).  By the score, not
    // the weight: a token that is seen gives its NaN whatever its weight.
    auto hidden = [&](float score) { return NB > 1 && !whole && score == -INFINITY; };
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const float ref = m[nb] == -INFINITY ? 0.0f : m[nb];
      float v[2][2][G], most[G] = {};
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float p = ex2(x[nb][tt][i] - ref);
          l[nb] += p;
#pragma unroll
          for (int gi = 0; gi < G; ++gi) {
            pm[nb][gi] = fmaf(p, hidden(x[nb][tt][i]) ? 0.0f : fmaf(8.0f, vs[tt][i][gi], vm[tt][i][gi]), pm[nb][gi]);
            v[tt][i][gi] = hidden(x[nb][tt][i]) ? 0.0f : p * vs[tt][i][gi];
            most[gi] = fmaxf(most[gi], v[tt][i][gi]);
          }
        }
      // Each group has a unit of its own: a group of small values beside one of large values keeps its
      // bits.  Only the exponents count, so that two groups' largest travel in the halves of a word.
      uint32_t tops = G == 2 ? __byte_perm(__float_as_uint(most[0]), __float_as_uint(most[G - 1]), 0x7632) : __float_as_uint(most[0]) >> 16;
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) tops = __vmaxu2(tops, __shfl_xor_sync(0xffffffffu, tops, off));
      // scaled so that the largest is in [2^21, 2^22); added to 2^23, the integer stands in the low bits
      float up[G];
#pragma unroll
      for (int gi = 0; gi < G; ++gi) {
        const int field = max(22, (int)(gi ? tops >> 23 : (tops >> 7) & 255u));
        up[gi] = __int_as_float((275 - field) << 23);
        f[nb][gi] = __int_as_float((field - 21) << 23);
      }
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int gi = 0; gi < G; ++gi) {
          const uint32_t v0 = __float_as_uint(fmaf(v[tt][0][gi], up[gi], 8388608.0f)), v1 = __float_as_uint(fmaf(v[tt][1][gi], up[gi], 8388608.0f));
          pb[nb][gi][0][tt] = transpose_8x8(__byte_perm(v0, v1, 0x5140));
          pb[nb][gi][1][tt] = transpose_8x8(__byte_perm(v0, v1, 0x7362));  // its second column is not used
        }
    }
#pragma unroll
    for (int gi = 0; gi < G; ++gi) {
      uint32_t vw[2][4];
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        const uint4 u = *reinterpret_cast<const uint4*>(stage + tt * S::TILE + KV_TILE * (HD / 2) + gi * 512 + t * 128 + ((g ^ (2 * t)) << 4));
        vw[tt][0] = u.x, vw[tt][1] = u.y, vw[tt][2] = u.z, vw[tt][3] = u.w;
      }
      int minus[NB][2][4];  // -8 times the sums of the weights' digits
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int k = 0; k < 2; ++k) mma_s8u8_zero(minus[nb][k], 0xF8F8F8F8u, pb[nb][gi][k][0], pb[nb][gi][k][1]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // channels 8 g + 2 i and 2 i + 1 of the group
        const uint32_t a0 = vw[0][i] & nib, a1 = (vw[0][i] >> 4) & nib, a2 = vw[1][i] & nib, a3 = (vw[1][i] >> 4) & nib;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          int d[2][4];
#pragma unroll
          for (int k = 0; k < 2; ++k) mma_u8u8(d[k], a0, a1, a2, a3, pb[nb][gi][k][0], pb[nb][gi][k][1], minus[nb][k]);
#pragma unroll
          for (int c = 0; c < 2; ++c)
            o[nb][4 * gi + i][c] = fmaf((float)(d[1][2 * c] * 65536 + d[0][2 * c + 1] * 256 + d[0][2 * c]), f[nb][gi], o[nb][4 * gi + i][c]);
        }
      }
    }
    __syncwarp();  // every lane has read the stage
    if (n + KVA_STAGES < mine) issue(n + KVA_STAGES, st);
    if (++st == KVA_STAGES) st = 0, phase ^= 1;
  }
  if (!fine) {  // given up: no copy may be in flight when the rings are used again
    if (lane == 0)
      for (int i = 0; i < KVA_STAGES; ++i) wait_drain(bars + 8 * i, 0, a.wait_cap_ns), wait_drain(bars + 8 * i, 1, a.wait_cap_ns);
    __syncwarp();
  }
  // join the warps
  __syncthreads();
  float* wout = reinterpret_cast<float*>(smem) + (size_t)warp * ROWS * S::OUT_LD;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
      l[nb] += __shfl_xor_sync(0xffffffffu, l[nb], off);
#pragma unroll
      for (int gi = 0; gi < G; ++gi) pm[nb][gi] += __shfl_xor_sync(0xffffffffu, pm[nb][gi], off);
    }
#pragma unroll
    for (int gi = 0; gi < G; ++gi)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float(&d0)[2] = o[nb][4 * gi + 2 * half];
        const float(&d1)[2] = o[nb][4 * gi + 2 * half + 1];
        *reinterpret_cast<float4*>(wout + (4 * nb + t) * S::OUT_LD + 64 * gi + 8 * g + 4 * half) =
            make_float4(d0[0] + pm[nb][gi], d0[1] + pm[nb][gi], d1[0] + pm[nb][gi], d1[1] + pm[nb][gi]);
      }
    if (g == 0) {
      // a row of NaN scores has no maximum, but its sum is NaN and has to come through
      ml[warp * 2 * ROWS + 4 * nb + t] = m[nb] > -INFINITY ? m[nb] : l[nb] == l[nb] ? -INFINITY : 0.0f;
      ml[warp * 2 * ROWS + ROWS + 4 * nb + t] = l[nb];
    }
  }
  __syncthreads();
  float* cout = reinterpret_cast<float*>(smem) + KVA_WARPS * ROWS * S::OUT_LD;
  constexpr int QUADS = HD / 4;  // four outputs at a time
  auto put = [&](int r, int c, float4 y, float sum, bool none) {
    const int q = row0 + r;
    const float by = none ? 0.0f : 1.0f / sum;
    st_f4(a.out + ((int64_t)b * a.q_len + q / per_kv) * a.ldo + (int64_t)(kvh * per_kv + q % per_kv) * HD + c,
          none ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(y.x * by, y.y * by, y.z * by, y.w * by), a.vec_out != 0);
  };
  for (int i = threadIdx.x; i < ROWS * QUADS; i += KVA_THREADS) {
    const int r = i / QUADS, c = 4 * (i % QUADS);
    if (row0 + r >= rows) break;
    float top = -INFINITY, sum = 0.0f, mw[KVA_WARPS];
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < KVA_WARPS; ++w) mw[w] = ml[w * 2 * ROWS + r], top = fmaxf(top, mw[w]);
#pragma unroll
    for (int w = 0; w < KVA_WARPS; ++w) {
      if (mw[w] != -INFINITY) {  // with a weight of zero too: its NaN has to come through
        const float e = ex2(mw[w] - top);
        const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<float*>(smem) + (w * ROWS + r) * S::OUT_LD + c);
        sum = fmaf(e, ml[w * 2 * ROWS + ROWS + r], sum);
        y.x = fmaf(e, v.x, y.x), y.y = fmaf(e, v.y, y.y), y.z = fmaf(e, v.z, y.z), y.w = fmaf(e, v.w, y.w);
      }
    }
    if (splits == 1) {
      put(r, c, y, sum, top == -INFINITY);
    } else {
      *reinterpret_cast<float4*>(cout + r * S::OUT_LD + c) = y;
      if (c == 0) ml[KVA_WARPS * 2 * ROWS + r] = top, ml[KVA_WARPS * 2 * ROWS + ROWS + r] = sum;
    }
  }
  if (splits == 1) return;
  // join the CTAs of the cluster, each writing its share of the outputs
  cluster_sync();
  const uint32_t cout_s = sbase + KVA_WARPS * ROWS * S::OUT_LD * 4, ml_s = sbase + S::ML + KVA_WARPS * 2 * ROWS * 4;
  for (int i = rank * KVA_THREADS + threadIdx.x; i < ROWS * QUADS; i += splits * KVA_THREADS) {
    const int r = i / QUADS, c = 4 * (i % QUADS);
    if (row0 + r >= rows) break;
    float top = -INFINITY, sum = 0.0f, ms[8], ls[8];
    float4 v[8], y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      ms[s] = -INFINITY;
      if (s < splits) {
        ms[s] = ld_cluster_f32(mapa_shared(ml_s + r * 4, s));
        ls[s] = ld_cluster_f32(mapa_shared(ml_s + ROWS * 4 + r * 4, s));
        v[s] = ld_cluster_f4(mapa_shared(cout_s + (r * S::OUT_LD + c) * 4, s));
      }
    }
#pragma unroll
    for (int s = 0; s < 8; ++s) top = fmaxf(top, ms[s]);
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      if (ms[s] != -INFINITY) {
        const float e = ex2(ms[s] - top);
        sum = fmaf(e, ls[s], sum);
        y.x = fmaf(e, v[s].x, y.x), y.y = fmaf(e, v[s].y, y.y), y.z = fmaf(e, v[s].z, y.z), y.w = fmaf(e, v[s].w, y.w);
      }
    }
    put(r, c, y, sum, top == -INFINITY);
  }
  cluster_sync();  // no CTA leaves while others read its shared memory
}

}  // namespace envg
