// kv4.hip — the cache held in 4 bits: launches for a context's own use (kv4_* below, ctx.h) and the operators on device buffers of include/tgx.h
// (kernels/kv4.h).  The operators know no context: device and stream come with the call, nothing is allocated, nothing waits.
#include "ctx.h"
#include "kernels/kv4.h"

namespace {

thread_local char g_op_err[256] = "";

int op_err(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_op_err, sizeof g_op_err, fmt, ap);
  va_end(ap);
  return code;
}

// the call's device is current inside, the caller's again afterwards
struct OnDevice {
  int before = -1, rc = TGX_OK;
  explicit OnDevice(int device) {
    int cur = -1, n = 0;
    if (hipGetDevice(&cur) == hipSuccess && cur == device) return;
    if (hipGetDeviceCount(&n) != hipSuccess || n <= 0) { (void)hipGetLastError(); rc = op_err(TGX_ERR_DEVICE, "no HIP device visible"); return; }
    if (device < 0 || device >= n) { rc = op_err(TGX_ERR_INVALID, "device ordinal %d out of range [0,%d)", device, n); return; }
    if (hipSetDevice(device) != hipSuccess) { (void)hipGetLastError(); rc = op_err(TGX_ERR_DEVICE, "hipSetDevice(%d) failed", device); return; }
    before = cur;
  }
  ~OnDevice() { if (before >= 0) (void)hipSetDevice(before); }
};

int num_cus_of(int device) {
  static int cus[64];      // (every writer writes the same number)
  if (device < 0 || device >= 64) return 256;
  int n = __atomic_load_n(&cus[device], __ATOMIC_RELAXED);
  if (n > 0) return n;
  if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || n <= 0) { (void)hipGetLastError(); return 256; }
  __atomic_store_n(&cus[device], n, __ATOMIC_RELAXED);
  return n;
}

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? TGX_OK : op_err(TGX_ERR_DEVICE, "%s: %s", what, hipGetErrorString(e));
}

int kv4_dt(int tgx) { return tgx == TGX_BF16 ? tgx::DT_BF16 : tgx == TGX_F16 ? tgx::DT_F16 : tgx == TGX_F32 ? tgx::DT_F32 : -1; }

int check_cache(const tgx_kv4_cache* c, const tgx_kv4_batch* b, tgx::Kv4Args& a) {
  if (!c || !b) return op_err(TGX_ERR_INVALID, "null argument");
  if (c->head_dim != 64 && c->head_dim != 128) return op_err(TGX_ERR_UNSUPPORTED, "head_dim %d (64 and 128 are built)", c->head_dim);
  if (c->kv_heads < 1 || c->kv_heads > 4096) return op_err(TGX_ERR_INVALID, "kv_heads %d out of range", c->kv_heads);
  if (c->pages < 0 || c->pages > 0x7fffffff || c->seqs < 0 || c->table_len < 0 || c->table_stride < c->table_len || c->table_len > (0x7fffffff >> tgx::KV_BLOCK_SHIFT))
    return op_err(TGX_ERR_INVALID, "cache: pages / seqs / table sizes out of range");
  if (b->entries < 0 || b->entries > 65535 || b->tokens < 0 || b->tokens > 0x7fffffff || b->max_count < 0) return op_err(TGX_ERR_INVALID, "batch: entries / tokens / max_count out of range");
  if (!b->offsets && b->tokens != b->entries) return op_err(TGX_ERR_INVALID, "batch: %lld tokens of %d entries without offsets", (long long)b->tokens, b->entries);
  if (b->entries && ((!c->pool && c->pages) || (!c->table && c->seqs && c->table_len) || !b->start)) return op_err(TGX_ERR_INVALID, "null argument");      // (none of nothing: a pool without pages)
  if ((uintptr_t)c->pool & 15) return op_err(TGX_ERR_INVALID, "the pool is not aligned to 16 bytes");
  a.pool = (unsigned int*)c->pool; a.pages = c->pages; a.table = c->table; a.table_stride = c->table_stride; a.table_len = c->table_len; a.seqs = c->seqs;
  a.kv_heads = c->kv_heads;
  a.entries = b->entries; a.max_count = b->offsets ? (int)std::min<int64_t>(b->max_count, b->tokens) : std::min(b->max_count, 1); a.tokens = b->tokens;
  a.each = 1; a.seq = b->seq; a.start = b->start; a.offsets = b->offsets;
  return TGX_OK;
}

int check_rows(const tgx_kv4_rows* r, const char* name) {
  if (!r || !r->data) return op_err(TGX_ERR_INVALID, "%s: null argument", name);
  if (kv4_dt(r->dtype) < 0) return op_err(TGX_ERR_INVALID, "%s: unknown dtype %d", name, r->dtype);
  if ((uintptr_t)r->data % (r->dtype == TGX_F32 ? 4 : 2)) return op_err(TGX_ERR_INVALID, "%s: not aligned to its elements", name);
  return TGX_OK;
}

int check_kv(const tgx_kv4_rows* k, const tgx_kv4_rows* v, tgx::Kv4Args& a) {
  int rc;
  if ((rc = check_rows(k, "k")) || (rc = check_rows(v, "v"))) return rc;
  if (k->dtype != v->dtype) return op_err(TGX_ERR_INVALID, "k and v have different dtypes");
  a.k = k->data; a.v = v->data; a.kv_dt = kv4_dt(k->dtype); a.k_ts = k->token_stride; a.k_hs = k->head_stride; a.v_ts = v->token_stride; a.v_hs = v->head_stride;
  return TGX_OK;
}

// outputs whose tokens or heads lie on each other would hold whichever was written last
int check_apart(const tgx_kv4_rows* r, const char* name, int64_t tokens, int heads) {
  if ((tokens > 1 && !r->token_stride) || (heads > 1 && !r->head_stride)) return op_err(TGX_ERR_INVALID, "%s: tokens or heads share memory (a stride of 0)", name);
  return TGX_OK;
}

// blocks of 32 positions that an entry of n tokens may touch
int blocks_of(int n) { return (n + 30) / 32 + 1; }

}  // namespace

// Few tokens a wave a (token, head), beyond 512 such waves a workgroup a block of 32 positions.  us tokens / blocks: one row, eight heads of 128, 16 tokens 4.0 / 4.8, 64 5.4 / 5.2, 512
// 15.1 / 4.9; 16 rows, 2 4.4 / 5.1, 5 5.0 / 5.2, 16 7.5 / 5.3, 2048 461 / 34
void kv4_launch_append(const tgx::Kv4Args& a, int hd, hipStream_t s) {
  if (!a.entries || !a.max_count) return;
  if (a.max_count == 1 || (long long)a.max_count * a.entries * a.kv_heads <= 512) {
    const dim3 grid(a.kv_heads, a.max_count, a.entries);
    if (hd == 64) hipLaunchKernelGGL(tgx::kv4_append_token_kernel<64>, grid, dim3(64), 0, s, a);
    else hipLaunchKernelGGL(tgx::kv4_append_token_kernel<128>, grid, dim3(64), 0, s, a);
    return;
  }
  const dim3 grid(a.kv_heads, blocks_of(a.max_count), a.entries);
  TGX_DT_SWITCH(a.kv_dt,
    if (hd == 64) hipLaunchKernelGGL((tgx::kv4_append_block_kernel<64, DT>), grid, dim3(128), 0, s, a);
    else hipLaunchKernelGGL((tgx::kv4_append_block_kernel<128, DT>), grid, dim3(256), 0, s, a);)
}

void kv4_launch_read(const tgx::Kv4Args& a, int hd, hipStream_t s) {
  if (!a.entries || !a.max_count) return;
  const dim3 grid(a.kv_heads, blocks_of(a.max_count), a.entries);
  TGX_DT_SWITCH(a.kv_dt,
    if (hd == 64) hipLaunchKernelGGL((tgx::kv4_read_kernel<64, DT>), grid, dim3(64), 0, s, a);
    else hipLaunchKernelGGL((tgx::kv4_read_kernel<128, DT>), grid, dim3(64), 0, s, a);)
}

// STEPS: single tokens of a model's rows, and nothing else
template <int HD, int QT, int TQ, int TP, bool STEPS>
static void launch_attend(const tgx::Kv4Args& a, const tgx::Kv4Plan& p, hipStream_t s) {
  const dim3 grid(a.kv_heads * p.splits, p.tiles, a.entries);
  const size_t lds = (size_t)p.kw * std::min<long long>(16, (long long)a.max_count * a.group) * HD * 4;
  if (a.max_count == 1 && a.group <= 4) {
    if (p.kw == 8) hipLaunchKernelGGL((tgx::kv4_attend_token_kernel<HD, 4, 8, QT, TQ, TP>), grid, dim3(512), lds, s, a);
    else hipLaunchKernelGGL((tgx::kv4_attend_token_kernel<HD, 4, 4, QT, TQ, TP>), grid, dim3(256), lds, s, a);
  } else if (a.max_count == 1 && a.group <= 8) {
    if (p.kw == 8) hipLaunchKernelGGL((tgx::kv4_attend_token_kernel<HD, 8, 8, QT, TQ, TP>), grid, dim3(512), lds, s, a);
    else hipLaunchKernelGGL((tgx::kv4_attend_token_kernel<HD, 8, 4, QT, TQ, TP>), grid, dim3(256), lds, s, a);
  } else if (p.kw == 4 && p.nt == 1) hipLaunchKernelGGL((tgx::kv4_attend_keys_kernel<HD, 1, 4, QT, TQ, TP>), grid, dim3(256), lds, s, a);
  else if constexpr (!STEPS) {
    if (p.kw == 4) hipLaunchKernelGGL((tgx::kv4_attend_keys_kernel<HD, 2, 4, QT, TQ, TP>), grid, dim3(256), lds, s, a);
    else hipLaunchKernelGGL((tgx::kv4_attend_columns_kernel<HD, 2, QT, TQ, TP>), grid, dim3(256), 0, s, a);
  }
}

// a.splits, a.part, a.ml follow from the plan and the workspace here.  Keys and values to append: a single token's join in the attention launch, where an entry is its sequence's only one
// (3 us less than a launch of its own); entries that name their sequences or bring several tokens may read what others bring, and an append launch comes first
void kv4_launch_attend(tgx::Kv4Args a, const tgx::Kv4Plan& p, int hd, float* ws, hipStream_t s) {
  if (!a.entries || !a.max_count) return;
  if (a.k && (a.max_count > 1 || a.seq || a.offsets)) { kv4_launch_append(a, hd, s); a.k = a.v = nullptr; }
  const size_t rows = (size_t)a.tokens * a.heads;
  a.splits = p.splits;
  a.part = ws; a.ml = ws + rows * p.splits * hd;
  // terms of queries and weights by the outputs' type (kernels/kv4.h)
  auto launch = [&](auto hd_c) {
    constexpr int HD = decltype(hd_c)::value;
    if (a.q_dt == tgx::DT_BF16) launch_attend<HD, tgx::DT_BF16, 1, 2, false>(a, p, s);
    else if (a.q_dt == tgx::DT_F16) launch_attend<HD, tgx::DT_F16, 2, 2, false>(a, p, s);
    else if (a.steps && a.max_count == 1) launch_attend<HD, tgx::DT_F32, 2, 2, true>(a, p, s);
    else launch_attend<HD, tgx::DT_F32, 3, 3, false>(a, p, s);
  };
  if (hd == 64) launch(std::integral_constant<int, 64>{});
  else launch(std::integral_constant<int, 128>{});
  if (p.splits > 1) {
    const dim3 grid(a.heads, a.max_count, a.entries);
    TGX_DT_SWITCH(a.q_dt,
      if (hd == 64) hipLaunchKernelGGL((tgx::kv4_combine_kernel<64, DT>), grid, dim3(256), 0, s, a);
      else hipLaunchKernelGGL((tgx::kv4_combine_kernel<128, DT>), grid, dim3(256), 0, s, a);)
  }
}

void launch_copy_pages(const tgx::CopyPagesArgs& a, int layers, hipStream_t s) {
  if (!a.n || !layers || !a.page) return;
  hipLaunchKernelGGL(tgx::copy_pages_kernel, dim3((unsigned)((a.page + tgx::COPY_PIECE - 1) / tgx::COPY_PIECE), a.n, layers), dim3(256), 0, s, a);
}

// ---- a context's cache in 4 bits (ctx.h) ----------------------------------------------------------------------------------------------------------------
namespace {

// table of rows whose every entry names one block of their own (steps), or runs of blocks (prompts): row b, entry i -> b * per + min(i, per - 1)
__global__ __launch_bounds__(256) void stage_tbl_kernel(int* tbl, int stride, int per) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < stride) tbl[(size_t)blockIdx.y * stride + i] = blockIdx.y * per + (i < per ? i : per - 1);
}

// the pages of layer l through the tables of rows that start at `tbl`
tgx::Kv4Args layer_args(const tgx_ctx* c, int l, const int* tbl, int rows) {
  tgx::Kv4Args a{};
  a.kv_heads = c->d.kv_heads;
  a.pool = c->kv4_pool + (size_t)l * c->kv_nblocks * tgx::kv4_page_words(a.kv_heads, c->d.head_dim);
  a.pages = c->kv_nblocks;
  a.table = tbl; a.table_stride = a.table_len = c->kv_tbl_stride; a.seqs = rows;
  a.kv_dt = c->dt;
  return a;
}

}  // namespace

int kv4_alloc(tgx_ctx* c) {
  const tgx_model_desc& d = c->d;
  const size_t B = (size_t)d.max_batch, words = (size_t)d.layers * c->kv_nblocks * tgx::kv4_page_words(d.kv_heads, d.head_dim);
  int rc;
  if ((rc = dev_alloc(c, &c->kv4_pool, words))) return rc;
  HIP_OK(c, hipMemset(c->kv4_pool, 0, words * 4));
  if ((rc = dev_alloc(c, &c->kv4_stage_tbl, B * (size_t)c->kv_tbl_stride)) || (rc = dev_alloc(c, &c->kv4_prompt_tbl, B * (size_t)c->kv_tbl_stride)) || (rc = dev_alloc(c, &c->kv4_zero, 1))) return rc;
  HIP_OK(c, hipMemset(c->kv4_zero, 0, 4));
  hipLaunchKernelGGL(stage_tbl_kernel, dim3((c->kv_tbl_stride + 255) / 256, (unsigned)B), dim3(256), 0, c->stream, c->kv4_stage_tbl, c->kv_tbl_stride, 1);
  HIP_OK(c, hipGetLastError());
  c->kv4_ws_floats = tgx::kv4_step_floats(d.max_batch, d.heads, d.kv_heads, d.head_dim, d.max_ctx, c->num_cus);
  return c->kv4_ws_floats ? dev_alloc(c, &c->kv4_ws, c->kv4_ws_floats) : TGX_OK;
}

int kv4_prompt_begin(tgx_ctx* c, int row0, int NB, int S) {
  const size_t per = (size_t)(S + tgx::KV_BLOCK - 1) / tgx::KV_BLOCK, need = per * (size_t)NB, block = (size_t)c->d.kv_heads * tgx::KV_BLOCK * c->d.head_dim * c->esz;
  if (need > c->kv4_prompt_blocks) {
    HIP_OK(c, hipStreamSynchronize(c->stream));
    if (c->kv4_pk) (void)hipFree(c->kv4_pk);
    if (c->kv4_pv) (void)hipFree(c->kv4_pv);
    c->kv4_pk = c->kv4_pv = nullptr; c->kv4_prompt_blocks = 0;
    int rc;
    if ((rc = dev_alloc(c, &c->kv4_pk, need * block)) || (rc = dev_alloc(c, &c->kv4_pv, need * block))) return rc;
    c->kv4_prompt_blocks = need;
    HIP_OK(c, hipMemsetAsync(c->kv4_pk, 0, need * block, c->stream));      // (a tile's tail behind the prompt is read and masked: numbers, as in a cache)
    HIP_OK(c, hipMemsetAsync(c->kv4_pv, 0, need * block, c->stream));
  }
  hipLaunchKernelGGL(stage_tbl_kernel, dim3((c->kv_tbl_stride + 255) / 256, NB), dim3(256), 0, c->stream, c->kv4_prompt_tbl, c->kv_tbl_stride, (int)per);
  for (int b = 0; b < NB; b++) {
    RowState& r = c->rows[(size_t)(row0 + b)];
    r.kcache = c->kv4_pk; r.vcache = c->kv4_pv; r.tbl = c->kv4_prompt_tbl + (size_t)b * c->kv_tbl_stride;
  }
  return TGX_OK;
}

void kv4_prompt_end(tgx_ctx* c, int row0, int NB) {
  for (int b = row0; b < row0 + NB; b++) {
    RowState& r = c->rows[(size_t)b];
    r.kcache = c->slab_k; r.vcache = c->slab_v; r.tbl = c->kv4_stage_tbl + (size_t)b * c->kv_tbl_stride;
  }
}

void kv4_prompt_append(tgx_ctx* c, int l, int row0, int NB, int S) {
  const long long hd = c->d.head_dim, per = (S + tgx::KV_BLOCK - 1) / tgx::KV_BLOCK;
  tgx::Kv4Args a = layer_args(c, l, c->rows[(size_t)row0].tbl4, NB);
  a.entries = NB; a.each = a.max_count = S; a.tokens = (long long)NB * S;
  a.start = c->rows[(size_t)row0].pos;                                  // (0: a prompt's pass moves them when it is through)
  a.k = c->kv4_pk; a.v = c->kv4_pv;
  a.k_hs = a.v_hs = tgx::KV_BLOCK * hd; a.slot_s = hd; a.block_s = c->d.kv_heads * tgx::KV_BLOCK * hd; a.entry_s = per * a.block_s;
  kv4_launch_append(a, (int)hd, c->stream);
}

// == append and flashAttention over keys [0, pos[row]] of R rows (Attention.h:103-112); one_sequence: the rows are positions of one sequence (a prompt by steps)
void kv4_step_attend(tgx_ctx* c, RowState* rv, int R, int l, bool one_sequence) {
  const tgx_model_desc& d = c->d;
  const long long hd = d.head_dim, qd = (long long)d.heads * hd;
  RowState& r = rv[0];
  tgx::Kv4Args a = layer_args(c, l, r.tbl4, R);
  if (one_sequence) a.table_stride = 0;
  a.entries = R; a.each = a.max_count = 1; a.tokens = R; a.start = r.pos;
  a.steps = 1;
  // the rows' staging blocks (positions of one sequence: places of one block)
  const long long block = d.kv_heads * tgx::KV_BLOCK * hd;
  ebyte *k = r.kcache, *v = r.vcache;
  if (one_sequence) { const long long row = (r.tbl4 - c->kv_tbl) / c->kv_tbl_stride; k += row * block * c->esz; v += row * block * c->esz; }
  else { const long long row = rv - c->rows.data(); k += row * block * c->esz; v += row * block * c->esz; }
  a.k = k; a.v = v; a.k_hs = a.v_hs = tgx::KV_BLOCK * hd; a.slot_s = hd; a.entry_s = one_sequence ? 0 : block;
  a.q = r.q; a.out = r.attn; a.q_dt = tgx::DT_F32; a.q_ts = a.o_ts = qd; a.q_hs = a.o_hs = hd;
  a.heads = d.heads; a.group = d.heads / d.kv_heads;
  tgx::kv4_scale(a, 1.0f / sqrtf((float)hd));
  a.act16 = c->act16 ? (c->dt == tgx::DT_BF16 ? 1 : 2) : 0;
  const tgx::Kv4Plan p = tgx::kv4_plan(R, 1, d.kv_heads, a.group, d.head_dim, 0, c->kv4_keys, c->num_cus);
  if (one_sequence) { kv4_launch_append(a, d.head_dim, c->stream); a.k = a.v = nullptr; }      // (a position reads what the others of the pass append)
  if (tgx::kv4_part_floats(p, a.tokens * d.heads, d.head_dim) > c->kv4_ws_floats) { c->launch_fault = "kv.bits 4: attention workspace"; return; }
  kv4_launch_attend(a, p, d.head_dim, c->kv4_ws, c->stream);
}

static int rows_copy(tgx_ctx* c, int row, int layer, float** tmp, size_t T, tgx::Kv4Args* a) {
  const size_t n = T * c->d.kv_heads * c->d.head_dim;
  if (hipMalloc((void**)tmp, 2 * n * 4) != hipSuccess) { (void)hipGetLastError(); return set_err(c, TGX_ERR_NOMEM, "%zu bytes of device memory", 2 * n * 4); }
  *a = layer_args(c, layer, c->rows[(size_t)row].tbl4, 1);
  a->entries = 1; a->each = a->max_count = (int)T; a->tokens = (long long)T; a->start = c->kv4_zero;
  a->k = *tmp; a->v = *tmp + n; a->kv_dt = tgx::DT_F32;
  a->k_ts = a->v_ts = (long long)c->d.kv_heads * c->d.head_dim; a->k_hs = a->v_hs = c->d.head_dim;
  return TGX_OK;
}
int kv4_read_rows(tgx_ctx* c, int row, int layer, float* k_out, float* v_out, size_t T) {
  if (!T) return TGX_OK;
  float* tmp = nullptr;
  tgx::Kv4Args a{};
  int rc = rows_copy(c, row, layer, &tmp, T, &a);
  if (rc) return rc;
  const size_t n = T * c->d.kv_heads * c->d.head_dim;
  kv4_launch_read(a, c->d.head_dim, c->stream);
  if (hipGetLastError() != hipSuccess) rc = set_err(c, TGX_ERR_DEVICE, "kv4 read");
  if (!rc && k_out) rc = copy_to_host(c, k_out, tmp, n * 4);
  if (!rc && v_out) rc = copy_to_host(c, v_out, tmp + n, n * 4);
  (void)hipStreamSynchronize(c->stream);
  (void)hipFree(tmp);
  return rc;
}
int kv4_write_rows(tgx_ctx* c, int row, int layer, const float* k_in, const float* v_in, size_t T) {
  if (!T) return TGX_OK;
  float* tmp = nullptr;
  tgx::Kv4Args a{};
  int rc = rows_copy(c, row, layer, &tmp, T, &a);
  if (rc) return rc;
  const size_t n = T * c->d.kv_heads * c->d.head_dim;
  hipError_t e = hipMemcpy(tmp, k_in, n * 4, hipMemcpyHostToDevice);
  if (e == hipSuccess) e = hipMemcpy(tmp + n, v_in, n * 4, hipMemcpyHostToDevice);
  if (e == hipSuccess) { kv4_launch_append(a, c->d.head_dim, c->stream); e = hipGetLastError(); }
  if (e == hipSuccess) e = hipStreamSynchronize(c->stream);
  (void)hipFree(tmp);
  return e == hipSuccess ? TGX_OK : set_err(c, TGX_ERR_DEVICE, "kv4 write: %s", hipGetErrorString(e));
}

extern "C" {

const char* tgx_op_last_error(void) { return g_op_err; }

int64_t tgx_kv4_page_bytes(int kv_heads, int head_dim) {
  if ((head_dim != 64 && head_dim != 128) || kv_heads < 1 || kv_heads > 4096) return -1;
  return (int64_t)tgx::kv4_page_words(kv_heads, head_dim) * 4;
}

int tgx_kv4_append(const tgx_kv4_cache* cache, const tgx_kv4_batch* batch, const tgx_kv4_rows* k, const tgx_kv4_rows* v, int device, void* stream) {
  tgx::Kv4Args a{};
  int rc;
  if ((rc = check_cache(cache, batch, a))) return rc;
  if (!a.entries || !a.max_count || !a.tokens) return TGX_OK;
  if ((rc = check_kv(k, v, a))) return rc;
  if (blocks_of(a.max_count) > 65535) return op_err(TGX_ERR_UNSUPPORTED, "max_count %d", a.max_count);
  OnDevice on(device);
  if (on.rc) return on.rc;
  kv4_launch_append(a, cache->head_dim, (hipStream_t)stream);
  return launched("kv4 append");
}

int tgx_kv4_read(const tgx_kv4_cache* cache, const tgx_kv4_batch* batch, const tgx_kv4_rows* k, const tgx_kv4_rows* v, int device, void* stream) {
  tgx::Kv4Args a{};
  int rc;
  if ((rc = check_cache(cache, batch, a))) return rc;
  if (!a.entries || !a.max_count || !a.tokens) return TGX_OK;
  if ((rc = check_kv(k, v, a)) || (rc = check_apart(k, "k", a.tokens, a.kv_heads)) || (rc = check_apart(v, "v", a.tokens, a.kv_heads))) return rc;
  if (blocks_of(a.max_count) > 65535) return op_err(TGX_ERR_UNSUPPORTED, "max_count %d", a.max_count);
  OnDevice on(device);
  if (on.rc) return on.rc;
  kv4_launch_read(a, cache->head_dim, (hipStream_t)stream);
  return launched("kv4 read");
}

static int attend_args(const tgx_kv4_cache* cache, const tgx_kv4_batch* batch, int heads, int window, int64_t max_keys, tgx::Kv4Args& a) {
  int rc;
  if ((rc = check_cache(cache, batch, a))) return rc;
  if (heads < 1 || heads % cache->kv_heads) return op_err(TGX_ERR_INVALID, "%d query heads over %d key / value heads", heads, cache->kv_heads);
  if (heads / cache->kv_heads > 16) return op_err(TGX_ERR_UNSUPPORTED, "GQA group size %d > 16", heads / cache->kv_heads);
  if (heads > 65535) return op_err(TGX_ERR_UNSUPPORTED, "%d query heads", heads);
  if (window < 0 || window > (1 << 30)) return op_err(TGX_ERR_INVALID, "window %d out of range", window);
  if (max_keys < 0 || max_keys > 0x7fffffff) return op_err(TGX_ERR_INVALID, "max_keys out of range");
  a.heads = heads; a.group = heads / cache->kv_heads; a.window = window;
  return TGX_OK;
}

int64_t tgx_kv4_attend_workspace(const tgx_kv4_cache* cache, const tgx_kv4_batch* batch, int heads, int window, int64_t max_keys, int device) {
  tgx::Kv4Args a{};
  if (attend_args(cache, batch, heads, window, max_keys, a)) return -1;
  if (!a.entries || !a.max_count || !a.tokens) return 0;
  const tgx::Kv4Plan p = tgx::kv4_plan(a.entries, a.max_count, a.kv_heads, a.group, cache->head_dim, window, max_keys, num_cus_of(device));
  return (int64_t)tgx::kv4_part_floats(p, a.tokens * heads, cache->head_dim) * 4;
}

int tgx_kv4_attend(const tgx_kv4_cache* cache, const tgx_kv4_batch* batch, const tgx_kv4_rows* q, int heads, const tgx_kv4_rows* k, const tgx_kv4_rows* v, float scale, int window,
                   int64_t max_keys, const tgx_kv4_rows* out, void* workspace, int64_t workspace_bytes, int device, void* stream) {
  tgx::Kv4Args a{};
  int rc;
  if ((rc = attend_args(cache, batch, heads, window, max_keys, a))) return rc;
  if (!a.entries || !a.max_count || !a.tokens) return TGX_OK;
  if ((rc = check_rows(q, "q")) || (rc = check_rows(out, "out")) || (rc = check_apart(out, "out", a.tokens, heads))) return rc;
  if (q->dtype != out->dtype) return op_err(TGX_ERR_INVALID, "q and out have different dtypes");
  if (!k != !v) return op_err(TGX_ERR_INVALID, "k and v come together");
  if (k && (rc = check_kv(k, v, a))) return rc;
  if (!std::isfinite(scale)) return op_err(TGX_ERR_INVALID, "scale is not finite");
  a.q = q->data; a.out = out->data; a.q_dt = kv4_dt(q->dtype); a.q_ts = q->token_stride; a.q_hs = q->head_stride; a.o_ts = out->token_stride; a.o_hs = out->head_stride;
  tgx::kv4_scale(a, scale);
  OnDevice on(device);
  if (on.rc) return on.rc;
  const tgx::Kv4Plan p = tgx::kv4_plan(a.entries, a.max_count, a.kv_heads, a.group, cache->head_dim, window, max_keys, num_cus_of(device));
  const int64_t need = (int64_t)tgx::kv4_part_floats(p, a.tokens * heads, cache->head_dim) * 4;
  if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))) return op_err(TGX_ERR_INVALID, "workspace: %lld bytes aligned to 16 are needed", (long long)need);
  // (the grids' second dimension: tiles of columns, tokens whose records are joined, blocks that are appended)
  if (p.tiles > 65535 || (p.splits > 1 && a.max_count > 65535) || (k && blocks_of(a.max_count) > 65535)) return op_err(TGX_ERR_UNSUPPORTED, "max_count %d", a.max_count);
  kv4_launch_attend(a, p, cache->head_dim, (float*)workspace, (hipStream_t)stream);
  return launched("kv4 attention");
}

int tgx_copy_pages(const void* src, int64_t src_pages, int64_t src_stride, void* dst, int64_t dst_pages, int64_t dst_stride, int layers, int64_t page_bytes, const int32_t* from,
                   const int32_t* to, int n, int device, void* stream) {
  if (n < 0 || n > 65535 || layers < 0 || layers > 65535) return op_err(TGX_ERR_INVALID, "%d pairs, %d layers (0 .. 65535)", n, layers);
  if (src_pages < 0 || dst_pages < 0 || page_bytes < 0 || src_stride < 0 || dst_stride < 0) return op_err(TGX_ERR_INVALID, "sizes out of range");
  if (!n || !layers || !page_bytes || !src_pages || !dst_pages) return TGX_OK;
  if (!src || !dst || !from || !to) return op_err(TGX_ERR_INVALID, "null argument");
  if (page_bytes % 16 || src_stride % 16 || dst_stride % 16 || ((uintptr_t)src & 15) || ((uintptr_t)dst & 15)) return op_err(TGX_ERR_INVALID, "pools, strides and pages are multiples of 16 bytes");
  if ((page_bytes + tgx::COPY_PIECE - 1) / tgx::COPY_PIECE > 0x7fffffff) return op_err(TGX_ERR_INVALID, "sizes out of range");
  if (layers > 1 && (dst_stride / page_bytes < dst_pages)) return op_err(TGX_ERR_INVALID, "dst: layers share memory (%lld bytes between them, %lld pages of %lld)", (long long)dst_stride, (long long)dst_pages, (long long)page_bytes);
  OnDevice on(device);
  if (on.rc) return on.rc;
  tgx::CopyPagesArgs a{};
  a.src = (const unsigned char*)src; a.dst = (unsigned char*)dst; a.src_pool = src_stride; a.dst_pool = dst_stride; a.page = page_bytes; a.src_pages = src_pages; a.dst_pages = dst_pages;
  a.from = from; a.to = to; a.n = n;
  launch_copy_pages(a, layers, (hipStream_t)stream);
  return launched("page copy");
}

}  // extern "C"
