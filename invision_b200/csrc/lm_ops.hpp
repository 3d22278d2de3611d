// lm_ops.hpp -- host side of the language-model decode operators (4-bit linears, q/k norm +
// rotation, the paged 4-bit cache and its attention).  Part of envgemm.cu's translation unit: it
// uses its device registry, error and launch helpers.
#pragma once

namespace {
constexpr uint32_t Q4_MAGIC = 0xE17A9E44u;
constexpr uint32_t KV4_MAGIC = 0xE17A9E4Cu;
constexpr int Q4_MAX_K = 57344;  // eight CTAs' shared memory holds four rows of x of this length
}  // namespace

struct envg_q4weight_s {
  uint32_t magic;
  int dev;
  uint8_t* d;
  size_t bytes;
  int layout;
  Q4View v;
};

struct envg_kv4_s {
  uint32_t magic;
  int dev;
  uint8_t* d;
  size_t bytes;
  int64_t pages;
  int page_size, kv_heads, head_dim;
};

namespace {

int lm_dev(Dev** d) {
  *d = cur();
  if (!*d) return fail(ENVG_ERR_STATE, "envg_init has not been called");
  return ENVG_OK;
}

int check_q4(Dev* d, envg_q4weight w) {
  if (!w || w->magic != Q4_MAGIC) return fail(ENVG_ERR_STATE, "invalid or freed 4-bit weight handle");
  if (w->dev != d->id) return fail(ENVG_ERR_STATE, "weight lives on device %d, current device is %d", w->dev, d->id);
  return ENVG_OK;
}

int check_kv4(Dev* d, envg_kv4 c) {
  if (!c || c->magic != KV4_MAGIC) return fail(ENVG_ERR_STATE, "invalid or freed cache handle");
  if (c->dev != d->id) return fail(ENVG_ERR_STATE, "cache lives on device %d, current device is %d", c->dev, d->id);
  return ENVG_OK;
}

bool f4_ok(const void* p, int64_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 4 == 0; }

// Device copies of a host-pointer call's operands, packed into one grow-only buffer.
class LmStage {
 public:
  explicit LmStage(Dev* d) : d_(d) {}
  // Reserves `bytes` and returns the piece's number; p() gives its address after commit().
  int add(size_t bytes) {
    at_.push_back(total_);
    total_ += (size_t)rup((int64_t)std::max<size_t>(bytes, 16), 256);
    return (int)at_.size() - 1;
  }
  int commit() { return ensure(d_, d_->lm, total_); }
  template <typename T>
  T* p(int i) const {
    return reinterpret_cast<T*>(reinterpret_cast<uint8_t*>(d_->lm.p) + at_[i]);
  }
  // rows x cols floats (or 4-byte integers) of row stride ld, packed
  int in(int i, const void* src, int64_t ld, int64_t rows, int64_t cols) {
    if (rows == 0 || cols == 0) return ENVG_OK;
    ENVG_CUDA(cudaMemcpy2DAsync(p<uint8_t>(i), cols * 4, src, ld * 4, cols * 4, rows, cudaMemcpyHostToDevice, stream_of(d_)));
    d_->st.h2d_bytes += 4.0 * rows * cols;
    return ENVG_OK;
  }
  int out(int i, void* dst, int64_t ld, int64_t rows, int64_t cols) {
    if (rows == 0 || cols == 0) return ENVG_OK;
    ENVG_CUDA(cudaMemcpy2DAsync(dst, ld * 4, p<uint8_t>(i), cols * 4, cols * 4, rows, cudaMemcpyDeviceToHost, stream_of(d_)));
    d_->st.d2h_bytes += 4.0 * rows * cols;
    return ENVG_OK;
  }

 private:
  Dev* d_;
  size_t total_ = 0;
  std::vector<size_t> at_;
};

int finish_call(Dev* d, int flags) {
  d->st.calls++;
  if (!(flags & ENVG_DEVICE_PTRS) || !(flags & ENVG_ASYNC)) return sync_and_check(d);
  return ENVG_OK;
}

// How a 4-bit linear is spread over the SMs (one CTA each): the cluster size, a power of two, that
// leaves the least work on the busiest CTA, counted in blocks plus a fixed cost per cluster
// exchange, among those whose part of x leaves room for a ring.
// Clusters of s CTAs that the GPU holds at once (they do not span its processor groups).
int q4_clusters(const Dev* d, int s) {
  static int held[64][4];
  int& n = held[d->id][s == 2 ? 1 : s == 4 ? 2 : s == 8 ? 3 : 0];
  if (s == 1) return d->sms;
  if (n > 0) return n;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(d->sms / s * s));
  cfg.blockDim = dim3(Q4_THREADS);
  cfg.dynamicSmemBytes = Q4_SMEM;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)s, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  cfg.attrs = at, cfg.numAttrs = 1;
  if (cudaFuncSetAttribute(k_q4<1, 128, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, Q4_SMEM) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, k_q4<1, 128, false>, &cfg) != cudaSuccess || n < 1) {
    cudaGetLastError();
    n = std::max(1, d->sms / (2 * s));
  }
  return n;
}

template <int NT, bool HALF>
bool q4_plan(const Dev* d, const Q4View& w, int M, Q4Plan* best) {
  using S = Q4Smem<NT, HALF>;
  double least = 0.0;
  bool found = false;
  for (int s = 1; s <= 8; s *= 2) {
    const int kb = (int)cdiv(w.kblocks, s);
    const int room = Q4_SMEM - S::FIXED - S::x_bytes(kb, w.group);
    int stages = room / (Q4_WARPS * q4_block_bytes(w.group));
    stages = stages >= 6 ? 6 : stages >= 4 ? 4 : stages;
    if (stages < 3 || kb * (s - 1) >= w.kblocks) continue;  // (every CTA has work)
    // the launch rows of more than MC rows of x share the GPU: one wave of CTAs with more tiles each
    // rather than several waves (a CTA's start costs as much as about 64 blocks)
    const int held = q4_clusters(d, s), chunks = (int)cdiv(M, S::MC);
    const int clusters = (int)std::min<int64_t>(w.tiles, std::max(1, held / chunks));
    const double waves = (double)cdiv((int64_t)clusters * chunks, held);
    const double cost = waves * ((double)cdiv(w.tiles, clusters) * kb / Q4_WARPS + 4.0 + (s > 1 ? 4.0 : 0.0));
    if (found && cost >= least) continue;
    least = cost, found = true;
    best->splits = s, best->log_splits = s == 1 ? 0 : s == 2 ? 1 : s == 4 ? 2 : 3, best->clusters = clusters, best->kb_per = kb, best->stages = stages;
    best->each = w.tiles / clusters, best->rest = w.tiles % clusters;
  }
  return found;
}

template <int NT, int GROUP, bool HALF>
int launch_q4_t(Dev* d, const Q4Args& a, const Q4Plan& p) {
  static bool attr_set[64] = {};
  if (!attr_set[d->id]) {
    ENVG_CUDA(cudaFuncSetAttribute(k_q4<NT, GROUP, HALF>, cudaFuncAttributeMaxDynamicSharedMemorySize, Q4_SMEM));
    attr_set[d->id] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.clusters * p.splits), (unsigned)cdiv(a.M, Q4Smem<NT, HALF>::MC));
  cfg.blockDim = dim3(Q4_THREADS);
  cfg.dynamicSmemBytes = Q4Smem<NT, HALF>::total(p.kb_per, p.stages, GROUP);
  cfg.stream = stream_of(d);
  cudaLaunchAttribute at[2];
  int n = 0;
  if (p.splits > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = (unsigned)p.splits, at[n].val.clusterDim.y = 1, at[n].val.clusterDim.z = 1;
    ++n;
  }
  if (d->pdl && !g_prof_on) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = (unsigned)n;
  ENVG_CUDA(cudaLaunchKernelEx(&cfg, k_q4<NT, GROUP, HALF>, a, p));
  d->st.kernel_launches++;
  return ENVG_OK;
}

template <int NT, bool HALF>
int launch_q4_n(Dev* d, const Q4Args& a, const Q4Plan& p) {
  switch (a.w.group) {
    case 32: return launch_q4_t<NT, 32, HALF>(d, a, p);
    case 64: return launch_q4_t<NT, 64, HALF>(d, a, p);
    default: return launch_q4_t<NT, 128, HALF>(d, a, p);
  }
}

int launch_q4(Dev* d, const Q4Args& a) {
  const double bytes = (double)a.w.tiles * a.w.kblocks * q4_block_bytes(a.w.group) + 4.0 * a.M * a.w.K + 4.0 * a.M * a.w.N;
  ProfScope ps(stream_of(d), KID_Q4, 2.0 * a.M * (double)a.w.N * (double)a.w.K, bytes);
  Q4Plan p{};
  p.vec = f4_ok(a.x, a.ldx);
  // 16, 8, 4 or 2 rows at a time: as many as there are, fewer where K leaves no room for their parts
  if (a.M > 8 && q4_plan<4, true>(d, a.w, a.M, &p)) return launch_q4_n<4, true>(d, a, p);
  if (a.M > 4 && q4_plan<2, true>(d, a.w, a.M, &p)) return launch_q4_n<2, true>(d, a, p);
  if (a.M > 2 && q4_plan<2, false>(d, a.w, a.M, &p)) return launch_q4_n<2, false>(d, a, p);
  if (q4_plan<1, false>(d, a.w, a.M, &p)) return launch_q4_n<1, false>(d, a, p);
  return fail(ENVG_ERR_UNSUPPORTED, "linear_q4: K=%lld is too long", (long long)a.w.K);
}

int launch_norm_rope(Dev* d, const NormRopeArgs& a) {
  const int all = a.heads + a.kv_heads;
  int lanes = 1;
  while (lanes * 8 < a.hd) lanes *= 2;
  const int64_t runs = cdiv(a.heads, NR_HEADS) + cdiv(a.kv_heads, NR_HEADS), blocks = cdiv(a.tokens * runs * lanes, 256);
  if (blocks * 256 > UINT32_MAX) return fail(ENVG_ERR_ARG, "qk_norm_rope: %lld tokens are too many", (long long)a.tokens);
  ProfScope ps(stream_of(d), KID_NORM_ROPE, 0.0, 8.0 * (double)a.tokens * all * a.hd + 4.0 * (double)a.tokens * a.hd);
  const dim3 g((unsigned)blocks), b(256);
  switch (lanes) {
    case 1: ENVG_TRY(launch_pdl(d, k_qk_norm_rope<1>, g, b, 0, a)); break;
    case 2: ENVG_TRY(launch_pdl(d, k_qk_norm_rope<2>, g, b, 0, a)); break;
    case 4: ENVG_TRY(launch_pdl(d, k_qk_norm_rope<4>, g, b, 0, a)); break;
    case 8: ENVG_TRY(launch_pdl(d, k_qk_norm_rope<8>, g, b, 0, a)); break;
    case 16: ENVG_TRY(launch_pdl(d, k_qk_norm_rope<16>, g, b, 0, a)); break;
    default: ENVG_TRY(launch_pdl(d, k_qk_norm_rope<32>, g, b, 0, a)); break;
  }
  d->st.kernel_launches++;
  return ENVG_OK;
}

// Checks shared by the calls that name tokens of a cache through a page table.  The call touches
// the new tokens, the `before` tokens in front of them and the first `sinks`: only the pages of
// those have to exist.
int check_kv_call(Dev* d, envg_kv4 c, const int32_t* table, int64_t table_stride, const int32_t* ctx_lens, int batch,
                  int q_len, int64_t before, int sinks, int flags, const char* what) {
  ENVG_TRY(check_kv4(d, c));
  if (batch < 0 || q_len < 0 || table_stride < 0) return fail(ENVG_ERR_ARG, "%s: batch %d, q_len %d, table stride %lld", what, batch, q_len, (long long)table_stride);
  if (table_stride * c->page_size > INT32_MAX)
    return fail(ENVG_ERR_ARG, "%s: a table row names %lld tokens (at most 2^31 - 1)", what, (long long)(table_stride * c->page_size));
  if (batch == 0 || q_len == 0) return ENVG_OK;
  if (!table || !ctx_lens) return fail(ENVG_ERR_ARG, "%s: table or ctx_lens is NULL", what);
  if ((int64_t)batch * q_len > INT32_MAX) return fail(ENVG_ERR_ARG, "%s: batch x q_len is too large", what);
  if (!(flags & ENVG_DEVICE_PTRS)) {
    for (int b = 0; b < batch; ++b) {
      const int64_t n = ctx_lens[b];
      if (n < 0 || n > table_stride * c->page_size)
        return fail(ENVG_ERR_ARG, "%s: ctx_lens[%d] = %lld does not fit the table (%lld pages of %d)", what, b, (long long)n,
                    (long long)table_stride, c->page_size);
      const int64_t first = std::max<int64_t>(0, n - q_len - before) / c->page_size;
      for (int64_t i = 0; i < cdiv(n, c->page_size); ++i) {
        if (i < first && i >= cdiv(sinks, c->page_size)) continue;
        const int32_t page = table[b * table_stride + i];
        if (page < 0 || page >= c->pages)
          return fail(ENVG_ERR_ARG, "%s: table[%d][%lld] = %d names no page (%lld pages)", what, b, (long long)i, page, (long long)c->pages);
      }
    }
  }
  return ENVG_OK;
}

Kv4View kv_view(Dev* d, envg_kv4 c, const int32_t* table, int64_t stride, const int32_t* lens) {
  Kv4View v{};
  v.base = c->d;
  v.pages = c->pages;
  v.page_size = c->page_size;
  v.kv_heads = c->kv_heads;
  v.page_tiles = FastDiv((uint32_t)(c->page_size / KV_TILE));
  v.table = table;
  v.table_stride = stride;
  v.ctx_lens = lens;
  v.status = d->d_status;
  return v;
}

// Append (k, v are read) or read back (k, v are written) the last q_len tokens of each sequence.
int kv4_rows(const envg_kv4_rows* r, int flags, bool read) {
  const char* what = read ? "kv4_read" : "kv4_append";
  Dev* d;
  ENVG_TRY(lm_dev(&d));
  if (!r) return fail(ENVG_ERR_ARG, "%s: NULL arguments", what);
  const envg_kv4 c = r->cache;
  float *k = r->k, *v = r->v;
  const int64_t ldk = r->ldk, ldv = r->ldv, stride = r->table_stride;
  const int32_t *table = r->table, *lens = r->ctx_lens;
  const int batch = r->batch, q_len = r->q_len;
  ENVG_TRY(check_kv_call(d, c, table, stride, lens, batch, q_len, 0, 0, flags, what));
  const int64_t rows = (int64_t)batch * q_len, width = (int64_t)c->kv_heads * c->head_dim;
  if (rows == 0) return ENVG_OK;
  if (!k || !v) return fail(ENVG_ERR_ARG, "%s: k or v is NULL", what);
  if (ldk < width || ldv < width) return fail(ENVG_ERR_ARG, "%s: a row stride is shorter than kv_heads x head_dim", what);
  if (read && k == v) return fail(ENVG_ERR_ARG, "kv4_read: k and v are the same buffer");
  LmStage st(d);
  const bool devp = (flags & ENVG_DEVICE_PTRS) != 0;
  float *dk = k, *dv = v;
  int64_t lk = ldk, lv = ldv;
  int ik = 0, iv = 0;
  if (!devp) {
    ik = st.add(rows * width * 4), iv = st.add(rows * width * 4);
    const int it = st.add(batch * stride * 4), il = st.add((size_t)batch * 4);
    ENVG_TRY(st.commit());
    if (!read) {
      ENVG_TRY(st.in(ik, k, ldk, rows, width));
      ENVG_TRY(st.in(iv, v, ldv, rows, width));
    }
    ENVG_TRY(st.in(it, table, stride, batch, stride));
    ENVG_TRY(st.in(il, lens, batch, 1, batch));
    dk = st.p<float>(ik), dv = st.p<float>(iv), lk = lv = width;
    table = st.p<int32_t>(it), lens = st.p<int32_t>(il);
  }
  KvRowsArgs a{};
  a.c = kv_view(d, c, table, stride, lens);
  a.k = dk, a.v = dv, a.ldk = lk, a.ldv = lv;
  a.hd = c->head_dim, a.batch = batch, a.q_len = q_len;
  // two or four tokens to a thread once they fill the GPU's threads all the same (append and read of
  // 1024 / 2048 / 4096 / 8192 / 16384 tokens, 8 heads of 128, us: 9.7 / 15.2 / 25.8 / - / - with one,
  // 10.3 / 14.5 / 23.9 / 40.9 / 78.2 with two, - / 18.2 / 25.6 / 42.4 / 75.8 with four)
  const int run_threads = c->kv_heads * 2 * (c->head_dim / KV_GROUP) * 8;
  const int64_t fill = rows * run_threads / ((int64_t)d->sms * 2048);
  const int each = q_len >= 4 && fill >= 10 ? 4 : q_len >= 2 && fill >= 1 ? 2 : 1;
  const int runs_seq = (int)cdiv(q_len, each);
  a.runs = batch * runs_seq;
  a.runs_per = std::max(1, 256 / run_threads);
  a.per_run = FastDiv((uint32_t)run_threads);
  a.seq = FastDiv((uint32_t)runs_seq);
  a.vec = f4_ok(dk, lk) && f4_ok(dv, lv);
  const dim3 grid((unsigned)cdiv(a.runs, a.runs_per), (unsigned)cdiv(run_threads, 256));
  {
    ProfScope ps(stream_of(d), read ? KID_KV4_READ : KID_KV4_APPEND, 0.0,
                 (double)rows * c->kv_heads * (8.0 * c->head_dim + c->head_dim + 8 * (c->head_dim / KV_GROUP)));
    void (*kernel)(const KvRowsArgs) = read ? (each == 4 ? k_kv4_rows<true, 4> : each == 2 ? k_kv4_rows<true, 2> : k_kv4_rows<true, 1>)
                                            : (each == 4 ? k_kv4_rows<false, 4> : each == 2 ? k_kv4_rows<false, 2> : k_kv4_rows<false, 1>);
    ENVG_TRY(launch_pdl(d, kernel, grid, dim3(256), 0, a));
    d->st.kernel_launches++;
  }
  if (!devp && read) {
    ENVG_TRY(st.out(ik, k, ldk, rows, width));
    ENVG_TRY(st.out(iv, v, ldv, rows, width));
  }
  return finish_call(d, flags);
}

// CTAs that share one (sequence, kv head, row tile), a power of two up to 8 (the portable cluster).
// A CTA costs about as much as eight units of two tiles a warp, so a GPU that is full takes more
// CTAs only while they keep that (measured, us: 16 sequences of 8192 to 16384 tokens, 128 groups:
// 119 / 72 / 63 / 57 at 1 / 2 / 4 / 8; 32 windows of 1024, 256 groups: 15.1 / 15.7 / 22 / 34); one that
// is not takes them down to one unit a warp (512 tokens, 8 groups: 7.0 / 6.9 / 6.0 / 6.0).
int kv4_splits(Dev* d, int64_t groups, int64_t tokens) {
  const int64_t units = cdiv(tokens, 2 * KV_TILE);
  int s = 1;
  while (s < 8) {
    const int64_t each = units / (2 * s * KVA_WARPS);  // units a warp keeps
    const bool more = groups * s < d->sms ? each >= 1 : groups * s * 2 <= (int64_t)d->sms * 8 && each >= 8;
    if (!more) break;
    s *= 2;
  }
  return s;
}

template <int HD, int NB>
int launch_kv4_attn_t(Dev* d, KvAttnArgs a, int splits) {
  using S = KvaSmem<HD, NB>;
  static bool attr_set[64] = {};
  if (!attr_set[d->id]) {
    ENVG_CUDA(cudaFuncSetAttribute(k_kv4_attn<HD, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::TOTAL));
    attr_set[d->id] = true;
  }
  const int64_t tiles = cdiv((int64_t)(a.heads / a.c.kv_heads) * a.q_len, S::ROWS) * a.c.kv_heads;
  if (tiles * splits > INT32_MAX || a.batch > 65535)
    return fail(ENVG_ERR_UNSUPPORTED, "attention_kv4: %d sequences of %lld row tiles are too many", a.batch, (long long)tiles);
  a.splits = splits, a.log_splits = splits == 1 ? 0 : splits == 2 ? 1 : splits == 4 ? 2 : 3;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(splits * tiles), (unsigned)a.batch);
  cfg.blockDim = dim3(KVA_THREADS);
  cfg.dynamicSmemBytes = S::TOTAL;
  cfg.stream = stream_of(d);
  cudaLaunchAttribute at[2];
  int n = 0;
  if (splits > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = (unsigned)splits, at[n].val.clusterDim.y = 1, at[n].val.clusterDim.z = 1;
    ++n;
  }
  if (d->pdl && !g_prof_on) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = (unsigned)n;
  ENVG_CUDA(cudaLaunchKernelEx(&cfg, k_kv4_attn<HD, NB>, a));
  d->st.kernel_launches++;
  return ENVG_OK;
}

int launch_kv4_attn(Dev* d, const KvAttnArgs& a, int max_ctx) {
  const int64_t rows = (int64_t)a.batch * a.q_len;
  const double seen = a.window > 0 ? std::min<double>(max_ctx, (double)a.window + a.sinks + a.q_len) : max_ctx;
  ProfScope ps(stream_of(d), KID_KV4_ATTN, 4.0 * a.hd * a.heads * (double)rows * seen,
               seen * a.batch * a.c.kv_heads * (a.hd + 8 * (a.hd / KV_GROUP)) + 8.0 * (double)rows * a.heads * a.hd);
  // rows that read one kv head: 4 or 8 at a time (16 took 255 registers and was no faster)
  const int64_t shared = (int64_t)(a.heads / a.c.kv_heads) * a.q_len;
  const bool four = shared <= 4;
  const int splits = kv4_splits(d, cdiv(shared, four ? 4 : 8) * a.c.kv_heads * a.batch, (int64_t)seen);
  if (a.hd == 128) return four ? launch_kv4_attn_t<128, 1>(d, a, splits) : launch_kv4_attn_t<128, 2>(d, a, splits);
  return four ? launch_kv4_attn_t<64, 1>(d, a, splits) : launch_kv4_attn_t<64, 2>(d, a, splits);
}

}  // namespace

extern "C" {

int envg_quantize_q4(const uint16_t* w_bf16, const float* w_f32, int64_t N, int64_t K, int group, uint8_t* codes,
                     float* scales, uint8_t* zeros) {
  if ((w_bf16 == nullptr) == (w_f32 == nullptr)) return fail(ENVG_ERR_ARG, "exactly one of w_bf16 / w_f32 must be set");
  if (N < 0 || K <= 0) return fail(ENVG_ERR_ARG, "quantize_q4: N=%lld K=%lld", (long long)N, (long long)K);
  if (group != 32 && group != 64 && group != 128) return fail(ENVG_ERR_ARG, "quantize_q4: group %d (32, 64 or 128)", group);
  if (N > 0 && (!codes || !scales || !zeros)) return fail(ENVG_ERR_ARG, "quantize_q4: NULL output");
  const WSrc src{w_bf16, w_f32, K};
  const int64_t ldc = (K + 1) / 2, ng = cdiv(K, group);
  for (int64_t n = 0; n < N; ++n)
    for (int64_t g = 0; g < ng; ++g) {
      const int64_t k0 = g * group, k1 = std::min<int64_t>(K, k0 + group);
      float lo = 0.0f, hi = 0.0f;  // the range always holds 0, so that 0 stays 0
      for (int64_t k = k0; k < k1; ++k) {
        const float v = src.value(n, k);
        if (!std::isfinite(v)) return fail(ENVG_ERR_ARG, "quantize_q4: W[%lld][%lld] is not finite", (long long)n, (long long)k);
        lo = std::min(lo, v), hi = std::max(hi, v);
      }
      const float s = std::isfinite(hi - lo) ? (hi - lo) / 15.0f : hi / 15.0f - lo / 15.0f;
      const int z = s > 0.0f ? (int)std::nearbyint(std::min(15.0f, std::max(0.0f, -lo / s))) : 8;
      scales[n * ng + g] = s;
      zeros[n * ng + g] = (uint8_t)z;
      for (int64_t k = k0; k < k1; ++k) {
        const float c = s > 0.0f ? std::nearbyint(src.value(n, k) / s) + z : 8.0f;
        const uint8_t q = (uint8_t)std::min(15.0f, std::max(0.0f, c));
        uint8_t& b = codes[n * ldc + (k >> 1)];
        b = (k & 1) ? (uint8_t)((b & 15) | (q << 4)) : q;
      }
    }
  return ENVG_OK;
}

int envg_weight_upload_q4(const uint8_t* codes, const float* scales, const uint8_t* zeros, int64_t N, int64_t K,
                          int group, int layout_flags, int flags, envg_q4weight* out) {
  std::lock_guard<std::recursive_mutex> lk(g_mu);
  if (!out) return fail(ENVG_ERR_ARG, "out handle pointer is NULL");
  *out = nullptr;
  Dev* d;
  ENVG_TRY(lm_dev(&d));
  if (!codes || !scales) return fail(ENVG_ERR_ARG, "weight_upload_q4: codes or scales is NULL");
  if (N <= 0 || K <= 0 || N > INT32_MAX / 2 || K > INT32_MAX / 2)
    return fail(ENVG_ERR_ARG, "weight_upload_q4: N=%lld K=%lld", (long long)N, (long long)K);
  if (K > Q4_MAX_K) return fail(ENVG_ERR_UNSUPPORTED, "weight_upload_q4: K=%lld (at most %d)", (long long)K, Q4_MAX_K);
  if (group != 32 && group != 64 && group != 128)
    return fail(ENVG_ERR_ARG, "weight_upload_q4: group %d (32, 64 or 128)", group);
  if (layout_flags != ENVG_LAYOUT_PLAIN && layout_flags != ENVG_LAYOUT_GATE_UP)
    return fail(ENVG_ERR_ARG, "weight_upload_q4: layout %d (PLAIN or GATE_UP)", layout_flags);
  const bool gu = layout_flags == ENVG_LAYOUT_GATE_UP;
  if (gu && N % 2) return fail(ENVG_ERR_ARG, "weight_upload_q4: a GATE_UP weight has an even number of rows");
  Q4View v{};
  v.tiles = (int)(gu ? cdiv(N / 2, 8) : cdiv(N, 16));
  v.kblocks = (int)cdiv(K, Q4_COLS);
  v.group = group, v.gate_up = gu ? 1 : 0, v.N = N, v.K = K;
  const int64_t blocks = (int64_t)v.tiles * v.kblocks;
  if (blocks > INT32_MAX) return fail(ENVG_ERR_ARG, "weight_upload_q4: N=%lld K=%lld is too large", (long long)N, (long long)K);
  const size_t bytes = (size_t)blocks * q4_block_bytes(group);
  const size_t cb = (size_t)N * ((K + 1) / 2), ng = (size_t)N * cdiv(K, group);
  uint8_t *dst = nullptr, *raw = nullptr;
  if (cudaMalloc(reinterpret_cast<void**>(&dst), bytes) != cudaSuccess) {
    cudaGetLastError();
    return fail(ENVG_ERR_OOM, "4-bit weight allocation of %zu bytes failed", bytes);
  }
  cudaStream_t s = stream_of(d);
  int rc = ENVG_OK;
  if (!(flags & ENVG_DEVICE_PTRS)) {
    const size_t so = (cb + 255) & ~size_t(255), zo = so + ng * 4;
    if (cudaMalloc(reinterpret_cast<void**>(&raw), zo + ng) != cudaSuccess) {
      cudaGetLastError();
      cudaFree(dst);
      return fail(ENVG_ERR_OOM, "4-bit weight staging of %zu bytes failed", zo + ng);
    }
    cudaError_t e = cudaMemcpyAsync(raw, codes, cb, cudaMemcpyHostToDevice, s);
    if (e == cudaSuccess) e = cudaMemcpyAsync(raw + so, scales, ng * 4, cudaMemcpyHostToDevice, s);
    if (e == cudaSuccess && zeros) e = cudaMemcpyAsync(raw + zo, zeros, ng, cudaMemcpyHostToDevice, s);
    if (e != cudaSuccess) rc = fail(ENVG_ERR_CUDA, "weight_upload_q4: copy failed: %s", cudaGetErrorString(e));
    d->st.h2d_bytes += (double)cb + 4.0 * ng + (zeros ? (double)ng : 0.0);
    codes = raw, scales = reinterpret_cast<const float*>(raw + so), zeros = zeros ? raw + zo : nullptr;
  }
  if (rc == ENVG_OK) {
    k_q4_pack<<<(unsigned)blocks, 256, 0, s>>>(v, dst, codes, scales, zeros, d->d_status);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) rc = fail(ENVG_ERR_CUDA, "k_q4_pack launch failed: %s", cudaGetErrorString(e));
    d->st.kernel_launches++;
  }
  const int rs = sync_and_check(d);
  if (rc == ENVG_OK) rc = rs;
  if (raw) cudaFree(raw);
  if (rc != ENVG_OK) {
    cudaFree(dst);
    return rc;
  }
  v.base = dst;
  envg_q4weight w = new envg_q4weight_s{};
  w->magic = Q4_MAGIC, w->dev = d->id, w->d = dst, w->bytes = bytes, w->layout = layout_flags, w->v = v;
  d->st.weight_bytes += bytes;
  *out = w;
  return ENVG_OK;
}

int envg_q4weight_free(envg_q4weight w) {
  std::lock_guard<std::recursive_mutex> lk(g_mu);
  if (!w || w->magic != Q4_MAGIC) return fail(ENVG_ERR_STATE, "invalid or already freed 4-bit weight handle");
  Dev* d = (w->dev >= 0 && w->dev < 64 && g_dev[w->dev].ready) ? &g_dev[w->dev] : nullptr;
  if (d) cudaStreamSynchronize(stream_of(d));
  cudaFree(w->d);  // waits for work on other streams that still reads it
  if (d) d->st.weight_bytes -= std::min<uint64_t>(d->st.weight_bytes, w->bytes);
  w->magic = 0;
  delete w;
  return ENVG_OK;
}

int envg_linear_q4(const envg_linear_q4_args* q, int flags) {
  std::lock_guard<std::recursive_mutex> lk(g_mu);
  Dev* d;
  ENVG_TRY(lm_dev(&d));
  if (!q) return fail(ENVG_ERR_ARG, "linear_q4: NULL arguments");
  float* dst = q->dst;
  const float *x = q->x, *bias = q->bias, *gate = q->gate;
  const envg_q4weight W = q->W;
  const int64_t ldd = q->ldd, ldx = q->ldx, M = q->M, K = q->K, N = q->N;
  const int epilogue = q->epilogue;
  ENVG_TRY(check_q4(d, W));
  if (K != W->v.K || N != W->v.N)
    return fail(ENVG_ERR_ARG, "linear_q4: [K=%lld, N=%lld] does not match the weight [N=%lld, K=%lld]", (long long)K,
                (long long)N, (long long)W->v.N, (long long)W->v.K);
  const bool gu = W->layout == ENVG_LAYOUT_GATE_UP;
  if ((epilogue == ENVG_EPI_SILU_GATE) != gu)
    return fail(ENVG_ERR_ARG, "linear_q4: SILU_GATE goes with (and only with) a GATE_UP weight");
  if (epilogue != ENVG_EPI_NONE && epilogue != ENVG_EPI_BIAS && epilogue != ENVG_EPI_SILU_GATE &&
      epilogue != ENVG_EPI_GATED_RESIDUAL)
    return fail(ENVG_ERR_ARG, "linear_q4: epilogue %d not valid for a linear", epilogue);
  if (epilogue == ENVG_EPI_BIAS && !bias) return fail(ENVG_ERR_ARG, "linear_q4: BIAS epilogue without bias");
  if (epilogue == ENVG_EPI_GATED_RESIDUAL && !gate) return fail(ENVG_ERR_ARG, "linear_q4: GATED_RESIDUAL without gate");
  if (M < 0 || M > 65535) return fail(ENVG_ERR_ARG, "linear_q4: M=%lld outside [0, 65535]", (long long)M);
  const int64_t n_out = gu ? N / 2 : N;
  if (M == 0) return ENVG_OK;
  if (ldx < K || ldd < n_out) return fail(ENVG_ERR_ARG, "linear_q4: a row stride is shorter than its row");
  if (!dst || !x) return fail(ENVG_ERR_ARG, "linear_q4: dst or x is NULL");
  if ((const void*)dst == (const void*)x) return fail(ENVG_ERR_ARG, "linear_q4: dst aliases x");
  Q4Args a{};
  a.w = W->v;
  a.x = x, a.dst = dst, a.ldx = ldx, a.ldd = ldd, a.M = (int)M;
  a.mode = gu ? Q4_SILU_GATE : epilogue == ENVG_EPI_GATED_RESIDUAL ? Q4_GATED_RES : Q4_PLAIN;
  a.bias = bias;
  a.gate = a.mode == Q4_GATED_RES ? gate : nullptr;
  LmStage st(d);
  const bool devp = (flags & ENVG_DEVICE_PTRS) != 0;
  int iy = 0;
  if (!devp) {
    const int ix = st.add(M * K * 4);
    iy = st.add(M * n_out * 4);
    const int ib = st.add(N * 4), ig = st.add(N * 4);
    ENVG_TRY(st.commit());
    ENVG_TRY(st.in(ix, x, ldx, M, K));
    if (a.mode == Q4_GATED_RES) ENVG_TRY(st.in(iy, dst, ldd, M, n_out));
    if (bias) ENVG_TRY(st.in(ib, bias, N, 1, N));
    if (a.gate) ENVG_TRY(st.in(ig, gate, N, 1, N));
    a.x = st.p<float>(ix), a.dst = st.p<float>(iy), a.ldx = K, a.ldd = n_out;
    a.bias = bias ? st.p<float>(ib) : nullptr;
    a.gate = a.gate ? st.p<float>(ig) : nullptr;
  }
  ENVG_TRY(launch_q4(d, a));
  d->st.flops += 2.0 * (double)M * (double)N * (double)K;
  if (!devp) ENVG_TRY(st.out(iy, dst, ldd, M, n_out));
  return finish_call(d, flags);
}

int envg_qk_norm_rope(const envg_qk_norm_rope_args* r, int flags) {
  std::lock_guard<std::recursive_mutex> lk(g_mu);
  Dev* d;
  ENVG_TRY(lm_dev(&d));
  if (!r) return fail(ENVG_ERR_ARG, "qk_norm_rope: NULL arguments");
  float *q_dst = r->q_dst, *k_dst = r->k_dst;
  const float *q = r->q, *k = r->k, *q_weight = r->q_weight, *k_weight = r->k_weight;
  const float *cos_table = r->cos_table, *sin_table = r->sin_table;
  const int64_t ldqd = r->ldqd, ldkd = r->ldkd, ldq = r->ldq, ldk = r->ldk;
  const int64_t table_rows = r->table_rows, pos0 = r->pos0, tokens = r->tokens;
  const int32_t* positions = r->positions;
  const int heads = r->heads, kv_heads = r->kv_heads, head_dim = r->head_dim, interleaved = r->interleaved;
  const float eps = r->eps;
  if (head_dim < 8 || head_dim > 256 || head_dim % 8)
    return fail(ENVG_ERR_UNSUPPORTED, "qk_norm_rope: head_dim %d (a multiple of 8 up to 256)", head_dim);
  if (tokens < 0 || heads < 0 || kv_heads < 0 || heads > 65535 || kv_heads > 65535)
    return fail(ENVG_ERR_ARG, "qk_norm_rope: %lld tokens, %d + %d heads", (long long)tokens, heads, kv_heads);
  if (!(eps >= 0.0f)) return fail(ENVG_ERR_ARG, "qk_norm_rope: eps must not be negative");
  if ((cos_table == nullptr) != (sin_table == nullptr)) return fail(ENVG_ERR_ARG, "qk_norm_rope: cos and sin go together");
  if (tokens == 0 || heads + kv_heads == 0) return ENVG_OK;
  if (tokens > INT32_MAX) return fail(ENVG_ERR_ARG, "qk_norm_rope: %lld tokens are too many", (long long)tokens);
  const int64_t wq = (int64_t)heads * head_dim, wk = (int64_t)kv_heads * head_dim;
  if ((heads && (!q || !q_dst)) || (kv_heads && (!k || !k_dst))) return fail(ENVG_ERR_ARG, "qk_norm_rope: NULL operand");
  if ((heads && (ldq < wq || ldqd < wq)) || (kv_heads && (ldk < wk || ldkd < wk)))
    return fail(ENVG_ERR_ARG, "qk_norm_rope: a row stride is shorter than its heads x head_dim");
  // with another stride a token's output would overwrite rows that are still to be read (host pointers: no
  // matter, the operands are copied)
  if ((flags & ENVG_DEVICE_PTRS) && tokens > 1 && ((heads && q_dst == q && ldqd != ldq) || (kv_heads && k_dst == k && ldkd != ldk)))
    return fail(ENVG_ERR_ARG, "qk_norm_rope: in place the row strides have to be equal");
  if (cos_table) {
    if (table_rows <= 0) return fail(ENVG_ERR_ARG, "qk_norm_rope: empty position table");
    if (!positions && (pos0 < 0 || pos0 + tokens > table_rows))
      return fail(ENVG_ERR_ARG, "qk_norm_rope: positions %lld..%lld outside the table's %lld rows", (long long)pos0,
                  (long long)(pos0 + tokens - 1), (long long)table_rows);
    if (positions && !(flags & ENVG_DEVICE_PTRS))
      for (int64_t i = 0; i < tokens; ++i)
        if (positions[i] < 0 || positions[i] >= table_rows)
          return fail(ENVG_ERR_ARG, "qk_norm_rope: positions[%lld] = %d outside the table's %lld rows", (long long)i,
                      positions[i], (long long)table_rows);
  }
  NormRopeArgs a{};
  a.qd = q_dst, a.kd = k_dst, a.q = q, a.k = k, a.ldqd = ldqd, a.ldkd = ldkd, a.ldq = ldq, a.ldk = ldk;
  a.wq = q_weight, a.wk = k_weight, a.cos = cos_table, a.sin = sin_table, a.table_rows = table_rows;
  a.positions = positions, a.pos0 = pos0, a.tokens = tokens;
  a.heads = heads, a.kv_heads = kv_heads, a.hd = head_dim, a.eps = eps, a.interleaved = interleaved ? 1 : 0;
  a.by_hd = 1.0f / (float)head_dim;
  a.q_runs = (int)cdiv(heads, NR_HEADS);
  a.per_token = FastDiv((uint32_t)(a.q_runs + cdiv(kv_heads, NR_HEADS)));
  a.status = d->d_status;
  LmStage st(d);
  const bool devp = (flags & ENVG_DEVICE_PTRS) != 0;
  int iq = 0, ik = 0;
  if (!devp) {
    const int64_t half = head_dim / 2;
    // with pos0 only its rows of the tables travel
    const int64_t r0 = positions ? 0 : pos0, rows = positions ? table_rows : tokens;
    iq = st.add(tokens * wq * 4), ik = st.add(tokens * wk * 4);
    const int iwq = st.add(head_dim * 4), iwk = st.add(head_dim * 4);
    const int ic = st.add(cos_table ? rows * half * 4 : 0), is = st.add(cos_table ? rows * half * 4 : 0);
    const int ip = st.add(positions ? tokens * 4 : 0);
    ENVG_TRY(st.commit());
    if (heads) ENVG_TRY(st.in(iq, q, ldq, tokens, wq));
    if (kv_heads) ENVG_TRY(st.in(ik, k, ldk, tokens, wk));
    if (q_weight) ENVG_TRY(st.in(iwq, q_weight, head_dim, 1, head_dim));
    if (k_weight) ENVG_TRY(st.in(iwk, k_weight, head_dim, 1, head_dim));
    if (cos_table) {
      ENVG_TRY(st.in(ic, cos_table + r0 * half, half, rows, half));
      ENVG_TRY(st.in(is, sin_table + r0 * half, half, rows, half));
      a.cos = st.p<float>(ic), a.sin = st.p<float>(is), a.table_rows = rows, a.pos0 = 0;
    }
    if (positions) ENVG_TRY(st.in(ip, positions, tokens, 1, tokens));
    a.q = a.qd = st.p<float>(iq), a.k = a.kd = st.p<float>(ik);
    a.ldq = a.ldqd = wq, a.ldk = a.ldkd = wk;
    a.wq = q_weight ? st.p<float>(iwq) : nullptr, a.wk = k_weight ? st.p<float>(iwk) : nullptr;
    a.positions = positions ? st.p<int32_t>(ip) : nullptr;
  }
  a.vec = (!heads || (f4_ok(a.q, a.ldq) && f4_ok(a.qd, a.ldqd))) && (!kv_heads || (f4_ok(a.k, a.ldk) && f4_ok(a.kd, a.ldkd))) &&
          f4_ok(a.wq, 0) && f4_ok(a.wk, 0) && f4_ok(a.cos, 0) && f4_ok(a.sin, 0);
  ENVG_TRY(launch_norm_rope(d, a));
  if (!devp) {
    if (heads) ENVG_TRY(st.out(iq, q_dst, ldqd, tokens, wq));
    if (kv_heads) ENVG_TRY(st.out(ik, k_dst, ldkd, tokens, wk));
  }
  return finish_call(d, flags);
}

int envg_kv4_create(int64_t pages, int page_size, int kv_heads, int head_dim, envg_kv4* out) {
  std::lock_guard<std::recursive_mutex> lk(g_mu);
  if (!out) return fail(ENVG_ERR_ARG, "out handle pointer is NULL");
  *out = nullptr;
  Dev* d;
  ENVG_TRY(lm_dev(&d));
  if (head_dim != 64 && head_dim != 128) return fail(ENVG_ERR_UNSUPPORTED, "kv4_create: head_dim %d (64 or 128)", head_dim);
  if (pages <= 0 || pages > INT32_MAX || kv_heads <= 0 || kv_heads > 1024)
    return fail(ENVG_ERR_ARG, "kv4_create: %lld pages, %d kv heads", (long long)pages, kv_heads);
  if (page_size < KV_TILE || page_size > 1024 || page_size % KV_TILE)
    return fail(ENVG_ERR_ARG, "kv4_create: page_size %d (a multiple of %d up to 1024)", page_size, KV_TILE);
  const size_t bytes = (size_t)pages * kv_heads * (page_size / KV_TILE) * kv_tile_bytes(head_dim);
  uint8_t* p = nullptr;
  if (cudaMalloc(reinterpret_cast<void**>(&p), bytes) != cudaSuccess) {
    cudaGetLastError();
    return fail(ENVG_ERR_OOM, "cache allocation of %zu bytes failed", bytes);
  }
  cudaError_t e = cudaMemsetAsync(p, 0, bytes, stream_of(d));
  if (e == cudaSuccess) e = cudaStreamSynchronize(stream_of(d));
  if (e != cudaSuccess) {
    cudaFree(p);
    return fail(ENVG_ERR_CUDA, "kv4_create: clearing the cache failed: %s", cudaGetErrorString(e));
  }
  envg_kv4 c = new envg_kv4_s{};
  c->magic = KV4_MAGIC, c->dev = d->id, c->d = p, c->bytes = bytes;
  c->pages = pages, c->page_size = page_size, c->kv_heads = kv_heads, c->head_dim = head_dim;
  *out = c;
  return ENVG_OK;
}

int envg_kv4_free(envg_kv4 c) {
  std::lock_guard<std::recursive_mutex> lk(g_mu);
  if (!c || c->magic != KV4_MAGIC) return fail(ENVG_ERR_STATE, "invalid or already freed cache handle");
  Dev* d = (c->dev >= 0 && c->dev < 64 && g_dev[c->dev].ready) ? &g_dev[c->dev] : nullptr;
  if (d) cudaStreamSynchronize(stream_of(d));
  cudaFree(c->d);  // waits for work on other streams that still uses it
  c->magic = 0;
  delete c;
  return ENVG_OK;
}

int envg_kv4_append(const envg_kv4_rows* rows, int flags) {
  std::lock_guard<std::recursive_mutex> lk(g_mu);
  return kv4_rows(rows, flags, false);
}

int envg_kv4_read(const envg_kv4_rows* rows, int flags) {
  std::lock_guard<std::recursive_mutex> lk(g_mu);
  return kv4_rows(rows, flags, true);
}

int envg_attention_kv4(const envg_attention_kv4_args* r, int flags) {
  std::lock_guard<std::recursive_mutex> lk(g_mu);
  Dev* d;
  ENVG_TRY(lm_dev(&d));
  if (!r) return fail(ENVG_ERR_ARG, "attention_kv4: NULL arguments");
  float* dst = r->dst;
  const float* q = r->q;
  const envg_kv4 cache = r->cache;
  const int32_t *table = r->table, *ctx_lens = r->ctx_lens;
  const int64_t ldo = r->ldo, ldq = r->ldq, table_stride = r->table_stride;
  const int batch = r->batch, q_len = r->q_len, max_ctx = r->max_ctx, heads = r->heads, window = r->window, sinks = r->sinks;
  const float scale = r->scale;
  if (window < 0 || sinks < 0) return fail(ENVG_ERR_ARG, "attention_kv4: window %d, sinks %d", window, sinks);
  ENVG_TRY(check_kv_call(d, cache, table, table_stride, ctx_lens, batch, q_len, window > 0 ? window - 1 : INT32_MAX,
                         window > 0 ? sinks : 0, flags, "attention_kv4"));
  if (heads <= 0 || heads % cache->kv_heads || heads > 65535)
    return fail(ENVG_ERR_ARG, "attention_kv4: %d heads over %d kv heads", heads, cache->kv_heads);
  if (max_ctx < 0) return fail(ENVG_ERR_ARG, "attention_kv4: max_ctx %d", max_ctx);
  if (!(scale > 0.0f)) return fail(ENVG_ERR_ARG, "attention_kv4: scale must be positive");
  const int64_t rows = (int64_t)batch * q_len, width = (int64_t)heads * cache->head_dim;
  if (rows == 0) return ENVG_OK;
  if (!dst || !q) return fail(ENVG_ERR_ARG, "attention_kv4: dst or q is NULL");
  if (ldo < width || ldq < width) return fail(ENVG_ERR_ARG, "attention_kv4: a row stride is shorter than heads x head_dim");
  if ((const void*)dst == (const void*)q) return fail(ENVG_ERR_ARG, "attention_kv4: dst aliases q");
  LmStage st(d);
  const bool devp = (flags & ENVG_DEVICE_PTRS) != 0;
  KvAttnArgs a{};
  a.q = q, a.out = dst, a.ldq = ldq, a.ldo = ldo;
  int io = 0;
  if (!devp) {
    const int iq = st.add(rows * width * 4), it = st.add(batch * table_stride * 4), il = st.add((size_t)batch * 4);
    io = st.add(rows * width * 4);
    ENVG_TRY(st.commit());
    ENVG_TRY(st.in(iq, q, ldq, rows, width));
    ENVG_TRY(st.in(it, table, table_stride, batch, table_stride));
    ENVG_TRY(st.in(il, ctx_lens, batch, 1, batch));
    a.q = st.p<float>(iq), a.out = st.p<float>(io), a.ldq = a.ldo = width;
    table = st.p<int32_t>(it), ctx_lens = st.p<int32_t>(il);
  }
  a.c = kv_view(d, cache, table, table_stride, ctx_lens);
  a.batch = batch, a.q_len = q_len, a.heads = heads, a.hd = cache->head_dim;
  a.sl2 = scale * 1.4426950408889634f;
  a.wait_cap_ns = d->wait_cap_ns;
  a.vec = f4_ok(a.q, a.ldq), a.vec_out = f4_ok(a.out, a.ldo);
  const int64_t most = table_stride * cache->page_size;
  a.window = window < most ? window : 0;  // a window over all that a table row names hides nothing
  a.sinks = (int)std::min<int64_t>(sinks, most);
  ENVG_TRY(launch_kv4_attn(d, a, (int)(max_ctx > 0 ? std::min<int64_t>(max_ctx, most) : most)));
  if (!devp) ENVG_TRY(st.out(io, dst, ldo, rows, width));
  return finish_call(d, flags);
}

}  // extern "C"
