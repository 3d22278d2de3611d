// kv4.cuh -- kernels of a language-model layer between its projections at decode time: the
// per-head RMS norm and position rotation of queries and keys, the paged 4-bit key/value cache,
// and attention over that cache.
//
// Cache format.  A token's key (and value) of one kv head is cut into groups of 64 channels.  A
// group holds m = fp16(min x), s = fp16((max x - min x) / 15) and codes
// c = clamp(rint((x - m) / s), 0, 15); it stands for the values m + s c.  The codes of 16 tokens
// lie together in one tile, tiles of a (page, kv head) follow one another:
//   tile = K codes [16][hd / 2 bytes] | V codes [16][hd / 2 bytes] | scales [16][2][hd / 64] half2 (s, m)
// A 32-bit word holds 8 consecutive channels 64 gi + 8 r + j (nibble j, r = 0..7).  In a K row,
// word (gi, r) stands at byte (r / 2) * hd / 8 + (2 gi + r % 2) * 4, so that lane t of a quad
// finds the words of its 16-channel pieces side by side; in a V row at byte r * hd / 16 + 4 gi.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

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
  const int32_t* table;     // [batch][table_stride] page ids
  int64_t table_stride;
  const int32_t* ctx_lens;  // [batch] tokens held, this call's q_len new ones among them
  int* status;
};

// Tokens of sequence b, held to what its row of the table can name.
ENVG_DEV int kv_len(const Kv4View& c, int b) {
  const int64_t most = c.table_stride * c.page_size;
  const int n = __ldg(c.ctx_lens + b);
  if (n < 0 || n > most) {
    kv_flag(c.status, SITE_KV_LEN);
    return n < 0 ? 0 : (int)most;
  }
  return n;
}

// Tile of token `pos` of sequence b and kv head h; nullptr where the table names no page.
ENVG_DEV uint8_t* kv_tile(const Kv4View& c, int b, int h, int pos, int tile_bytes) {
  const int32_t page = __ldg(c.table + (int64_t)b * c.table_stride + pos / c.page_size);
  if (page < 0 || page >= c.pages) {
    kv_flag(c.status, SITE_KV_PAGE);
    return nullptr;
  }
  const int64_t per_page = c.page_size / KV_TILE;
  return c.base + (((int64_t)page * c.kv_heads + h) * per_page + (pos % c.page_size) / KV_TILE) * tile_bytes;
}

ENVG_DEV float4 ld_f4(const float* p, bool vec) {
  if (vec) return *reinterpret_cast<const float4*>(p);
  return make_float4(p[0], p[1], p[2], p[3]);
}
ENVG_DEV void st_f4(float* p, float4 v, bool vec) {
  if (vec) {
    *reinterpret_cast<float4*>(p) = v;
  } else {
    p[0] = v.x, p[1] = v.y, p[2] = v.z, p[3] = v.w;
  }
}

// ---- norm of queries and keys per head + position rotation ------------------------------------
// y = rot(x w / sqrt(mean x^2 + eps)); rot turns the pair (a, b) of channels into
// (a cos - b sin, b cos + a sin).  A pair is (i, i + hd/2), or (2i, 2i + 1) when interleaved.
// One thread holds four pairs (8 channels) of one head, so that a head's pairs never leave their
// thread and the norm is one shuffle tree over hd / 8 threads (rounded up to a power of two).
struct NormRopeArgs {
  float *qd, *kd;
  const float *q, *k;
  int64_t ldqd, ldkd, ldq, ldk;
  const float *wq, *wk, *cos, *sin;
  int64_t table_rows;
  const int32_t* positions;
  int64_t pos0, tokens;
  int heads, kv_heads, hd;
  float eps;
  int interleaved, vec;
  int* status;
};

template <int LANES>
__global__ void __launch_bounds__(256) k_qk_norm_rope(const NormRopeArgs a) {
  griddep_wait();
  griddep_launch_dependents();
  const int all = a.heads + a.kv_heads;
  const int64_t item = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LANES;
  const int li = threadIdx.x % LANES;
  const int64_t tok = item / all;
  const int h = (int)(item - tok * all);
  const bool work = tok < a.tokens && 8 * li < a.hd;
  const bool isq = h < a.heads;
  const bool vec = a.vec != 0;
  float4 x0 = make_float4(0.f, 0.f, 0.f, 0.f), x1 = x0;
  const int i0 = a.interleaved ? 8 * li : 4 * li;                 // first channels of the thread
  const int i1 = a.interleaved ? 8 * li + 4 : a.hd / 2 + 4 * li;  // and the other four
  if (work) {
    const float* src = isq ? a.q + tok * a.ldq + (int64_t)h * a.hd : a.k + tok * a.ldk + (int64_t)(h - a.heads) * a.hd;
    x0 = ld_f4(src + i0, vec);
    x1 = ld_f4(src + i1, vec);
  }
  float ss = x0.x * x0.x;
  ss = fmaf(x0.y, x0.y, ss), ss = fmaf(x0.z, x0.z, ss), ss = fmaf(x0.w, x0.w, ss);
  ss = fmaf(x1.x, x1.x, ss), ss = fmaf(x1.y, x1.y, ss), ss = fmaf(x1.z, x1.z, ss), ss = fmaf(x1.w, x1.w, ss);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (!work) return;
  const float inv = 1.0f / sqrtf(ss / (float)a.hd + a.eps);
  const float* w = isq ? a.wq : a.wk;
  float4 w0 = make_float4(1.f, 1.f, 1.f, 1.f), w1 = w0;
  if (w) w0 = ld_f4(w + i0, vec), w1 = ld_f4(w + i1, vec);
  x0 = make_float4(x0.x * inv * w0.x, x0.y * inv * w0.y, x0.z * inv * w0.z, x0.w * inv * w0.w);
  x1 = make_float4(x1.x * inv * w1.x, x1.y * inv * w1.y, x1.z * inv * w1.z, x1.w * inv * w1.w);
  if (a.cos) {
    int64_t pos = a.positions ? (int64_t)__ldg(a.positions + tok) : a.pos0 + tok;
    if (pos < 0 || pos >= a.table_rows) {
      kv_flag(a.status, SITE_ROPE_POS);
      pos = pos < 0 ? 0 : a.table_rows - 1;
    }
    const float4 c = ld_f4(a.cos + pos * (a.hd / 2) + 4 * li, vec);
    const float4 s = ld_f4(a.sin + pos * (a.hd / 2) + 4 * li, vec);
    if (a.interleaved) {
      x0 = make_float4(x0.x * c.x - x0.y * s.x, x0.y * c.x + x0.x * s.x, x0.z * c.y - x0.w * s.y, x0.w * c.y + x0.z * s.y);
      x1 = make_float4(x1.x * c.z - x1.y * s.z, x1.y * c.z + x1.x * s.z, x1.z * c.w - x1.w * s.w, x1.w * c.w + x1.z * s.w);
    } else {
      const float4 p = x0;
      x0 = make_float4(p.x * c.x - x1.x * s.x, p.y * c.y - x1.y * s.y, p.z * c.z - x1.z * s.z, p.w * c.w - x1.w * s.w);
      x1 = make_float4(x1.x * c.x + p.x * s.x, x1.y * c.y + p.y * s.y, x1.z * c.z + p.z * s.z, x1.w * c.w + p.w * s.w);
    }
  }
  float* dst = isq ? a.qd + tok * a.ldqd + (int64_t)h * a.hd : a.kd + tok * a.ldkd + (int64_t)(h - a.heads) * a.hd;
  st_f4(dst + i0, x0, vec);
  st_f4(dst + i1, x1, vec);
}

// ---- cache: write and read ----------------------------------------------------------------------
// Eight threads hold one group of 64 channels, eight consecutive channels (one word of codes)
// each; the group's minimum and maximum are one shuffle tree.  Every rounding is IEEE (no
// contraction), so equal inputs give equal codes on any path that uses the formula.
ENVG_DEV uint32_t kv_k_word(int hd, int tok, int gi, int r) { return tok * (hd / 2) + (r >> 1) * (hd / 8) + (2 * gi + (r & 1)) * 4; }
ENVG_DEV uint32_t kv_v_word(int hd, int tok, int gi, int r) { return KV_TILE * (hd / 2) + tok * (hd / 2) + r * (hd / 16) + 4 * gi; }
ENVG_DEV uint32_t kv_scale_at(int hd, int tok, int v, int gi) { return KV_TILE * hd + (tok * 2 + v) * (hd / KV_GROUP) * 4 + gi * 4; }

struct KvRowsArgs {
  Kv4View c;
  float *k, *v;  // [batch * q_len, ld], read by the append and written by the read
  int64_t ldk, ldv, items;
  int hd, batch, q_len, vec;
};

template <bool READ>
__global__ void __launch_bounds__(256) k_kv4_rows(const KvRowsArgs a) {
  griddep_wait();
  griddep_launch_dependents();
  const int G = a.hd / KV_GROUP;
  const int64_t item = ((int64_t)blockIdx.x * 256 + threadIdx.x) / 8;
  const int r = threadIdx.x % 8;
  const bool work = item < a.items;
  int64_t n = work ? item : a.items - 1;
  const int gi = (int)(n % G);
  n /= G;
  const int isv = (int)(n & 1);
  n >>= 1;
  const int h = (int)(n % a.c.kv_heads);
  const int64_t row = n / a.c.kv_heads;
  const int b = (int)(row / a.q_len);
  const int pos = kv_len(a.c, b) - a.q_len + (int)(row % a.q_len);
  const int tile_bytes = kv_tile_bytes(a.hd);
  uint8_t* tile = pos >= 0 ? kv_tile(a.c, b, h, pos, tile_bytes) : nullptr;
  const int tok = pos >= 0 ? pos % KV_TILE : 0;
  const uint32_t word_at = isv ? kv_v_word(a.hd, tok, gi, r) : kv_k_word(a.hd, tok, gi, r);
  const uint32_t scale_at = kv_scale_at(a.hd, tok, isv, gi);
  float* rows = isv ? a.v + row * a.ldv : a.k + row * a.ldk;
  rows += (int64_t)h * a.hd + gi * KV_GROUP + 8 * r;
  const bool vec = a.vec != 0;
  if (READ) {
    if (!work) return;
    float x[8] = {};
    if (tile) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(tile + word_at);
      const float2 sm = __half22float2(*reinterpret_cast<const __half2*>(tile + scale_at));
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = fmaf(sm.x, (float)((w >> (4 * j)) & 15u), sm.y);
    }
    st_f4(rows, make_float4(x[0], x[1], x[2], x[3]), vec);
    st_f4(rows + 4, make_float4(x[4], x[5], x[6], x[7]), vec);
  } else {
    const float4 p0 = ld_f4(rows, vec), p1 = ld_f4(rows + 4, vec);
    const float x[8] = {p0.x, p0.y, p0.z, p0.w, p1.x, p1.y, p1.z, p1.w};
    float lo = x[0], hi = x[0];
    bool nan = x[0] != x[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) lo = fminf(lo, x[j]), hi = fmaxf(hi, x[j]), nan |= x[j] != x[j];
    int any = nan ? 1 : 0;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      any |= __shfl_xor_sync(0xffffffffu, any, o);
    }
    if (!work || !tile) return;
    if (any) lo = hi = __int_as_float(0x7fc00000);  // a group with a NaN holds NaN
    const float low = lo < -KV_HALF_MAX ? -KV_HALF_MAX : lo > KV_HALF_MAX ? KV_HALF_MAX : lo;
    const float step = __fdiv_rn(__fsub_rn(hi, lo), 15.0f);
    const __half2 sm = __halves2half2(__float2half_rn(step > KV_HALF_MAX ? KV_HALF_MAX : step), __float2half_rn(low));
    const float s = __low2float(sm), m = __high2float(sm);
    uint32_t w = 0;
    if (s > 0.0f) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float c = rintf(__fdiv_rn(__fsub_rn(x[j], m), s));
        w |= (uint32_t)fminf(fmaxf(c, 0.0f), 15.0f) << (4 * j);
      }
    }
    *reinterpret_cast<uint32_t*>(tile + word_at) = w;
    if (r == 0) *reinterpret_cast<__half2*>(tile + scale_at) = sm;
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
};

// One warp per (row, head); lane l holds channels 8l..8l+7 (l < hd / 8).
__global__ void __launch_bounds__(128) k_kv4_attn_simple(const KvAttnArgs a) {
  griddep_wait();
  griddep_launch_dependents();
  const int64_t item = (int64_t)blockIdx.x * 4 + threadIdx.x / 32;
  const int lane = threadIdx.x & 31;
  if (item >= (int64_t)a.batch * a.q_len * a.heads) return;
  const int h = (int)(item % a.heads);
  const int64_t row = item / a.heads;
  const int b = (int)(row / a.q_len);
  const int p = kv_len(a.c, b) - a.q_len + (int)(row % a.q_len);
  const int kvh = h / (a.heads / a.c.kv_heads);
  const bool on = lane < a.hd / 8;
  const int gi = lane / 8, r = lane % 8;
  float q[8] = {}, o[8] = {}, m = -INFINITY, l = 0.0f;
  if (on)
    for (int j = 0; j < 8; ++j) q[j] = a.q[row * a.ldq + (int64_t)h * a.hd + 8 * lane + j];
  const int tile_bytes = kv_tile_bytes(a.hd);
  for (int j = 0; j <= p; ++j) {
    if (a.window > 0 && j <= p - a.window && j >= a.sinks) {
      j = p - a.window;
      continue;
    }
    const uint8_t* tile = kv_tile(a.c, b, kvh, j, tile_bytes);
    if (!tile) continue;
    const int tok = j % KV_TILE;
    float s = 0.0f, v[8] = {};
    if (on) {
      const uint32_t wk = *reinterpret_cast<const uint32_t*>(tile + kv_k_word(a.hd, tok, gi, r));
      const uint32_t wv = *reinterpret_cast<const uint32_t*>(tile + kv_v_word(a.hd, tok, gi, r));
      const float2 ks = __half22float2(*reinterpret_cast<const __half2*>(tile + kv_scale_at(a.hd, tok, 0, gi)));
      const float2 vs = __half22float2(*reinterpret_cast<const __half2*>(tile + kv_scale_at(a.hd, tok, 1, gi)));
      for (int c = 0; c < 8; ++c) {
        s = fmaf(q[c], fmaf(ks.x, (float)((wk >> (4 * c)) & 15u), ks.y), s);
        v[c] = fmaf(vs.x, (float)((wv >> (4 * c)) & 15u), vs.y);
      }
    }
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    s *= a.sl2;
    const float top = fmaxf(m, s);
    const float scale = exp2f(m - top), e = exp2f(s - top);
    m = top;
    l = fmaf(l, scale, e);
    for (int c = 0; c < 8; ++c) o[c] = fmaf(o[c], scale, e * v[c]);
  }
  if (on)
    for (int c = 0; c < 8; ++c) a.out[row * a.ldo + (int64_t)h * a.hd + 8 * lane + c] = l > 0.0f ? o[c] / l : (l == l ? 0.0f : l);
}

}  // namespace envg
