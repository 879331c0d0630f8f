// kv4_plan.h — the cache held in 4 bits (kernels/kv4.h): its arguments, where a code lies, what a call's entry brings, which pages it reads and how its attention is
// divided, as plain arithmetic (no HIP call: tests go through it on the CPU, the kernels through the same functions).
#pragma once
#include <algorithm>
#include <cstddef>

#if defined(__HIPCC__)
#define TGX_KV4 __host__ __device__ __forceinline__
#else
#define TGX_KV4 inline
#endif

namespace tgx {

constexpr int KV4_PAGE = 128, KV4_PAGE_SHIFT = 7, KV4_BLK = 32;      // tokens of a page, of a block

struct Kv4Args {
  unsigned int* pool; long long pages;                        // pages of one layer
  const int* table; int table_stride, table_len, seqs;        // [seqs][table_stride], table_len entries of a row count; a page outside [0, pages) counts as one without tokens
  int kv_heads;
  int entries, max_count; long long tokens;                   // the batch: entries of consecutive tokens of a sequence each
  int each;                                                   // tokens of an entry where there are no offsets
  const int *seq, *start, *offsets;                           // seq: entry's table row (null: entry e is row e); start: position of its first token; offsets [entries + 1] into the tokens (or null)
  // keys and values that join (append), or that come out (read): (token, kv head, channel) at token * k_ts + head * k_hs + channel elements, and in a context's staging blocks (token strides
  // of 0) at entry * entry_s + position / KV4_PAGE * block_s + position % KV4_PAGE * slot_s further on
  void *k, *v; int kv_dt; long long k_ts, k_hs, v_ts, v_hs, slot_s, block_s, entry_s;
  // attention
  const void* q; void* out; int q_dt; long long q_ts, q_hs, o_ts, o_hs;
  int heads, group;
  float scale_log2, q_sign, gap;                              // |score scale| * log2(e) (1 for a scale of 0), the scale's sign, 8 / scale_log2: see kv4_scale
  int window;                                                 // > 0: position p sees keys p - window + 1 .. p
  int splits; float *part, *ml;                               // splits > 1: [token * heads + head][splits][HD] sums, [..][splits][2] (maximum, denominator)
  int steps;                                                  // a model's steps (host only): 32-bit queries in two terms
  int act16;                                                  // outputs rounded to the storage type: 0 no, 1 bf16, 2 fp16 (option act.round16 of a model)
};

// tokens, first token and position of entry e; count 0 where the entry names no sequence or its tokens are not all in the batch
struct Kv4Entry { int seq, start, count; long long tok0; };
TGX_KV4 Kv4Entry kv4_entry(const Kv4Args& a, int e) {
  Kv4Entry n;
  n.seq = a.seq ? a.seq[e] : e;
  n.start = a.start[e] < -(1 << 30) ? -(1 << 30) : a.start[e];
  const long long o0 = a.offsets ? a.offsets[e] : (long long)e * a.each, c = a.offsets ? a.offsets[e + 1] - o0 : a.each;
  n.tok0 = o0;
  n.count = (int)(c < a.max_count ? c : a.max_count);
  if (o0 < 0 || c < 0 || o0 + n.count > a.tokens || n.seq < 0 || n.seq >= a.seqs || n.start > 0x7fffffff - n.count) n.count = 0;
  return n;
}

// elements in front of channel 0 of a key (value) of entry e's token `tok` at `pos`
TGX_KV4 long long kv4_kv_at(const Kv4Args& a, int e, long long tok, int pos, int kvh, bool value) {
  return tok * (value ? a.v_ts : a.k_ts) + kvh * (value ? a.v_hs : a.k_hs) + e * a.entry_s + (pos >> KV4_PAGE_SHIFT) * a.block_s + (pos & (KV4_PAGE - 1)) * a.slot_s;
}

// the words of a page's head, or null where the table names no page
TGX_KV4 unsigned int* kv4_page(const Kv4Args& a, int seq, int b, int kvh, int hd) {
  if (b < 0 || b >= a.table_len) return nullptr;
  const int p = a.table[(long long)seq * a.table_stride + b];
  if (p < 0 || p >= a.pages) return nullptr;
  return a.pool + ((size_t)p * a.kv_heads + kvh) * (size_t)(36 * hd);
}
TGX_KV4 size_t kv4_page_words(int kv_heads, int hd) { return (size_t)kv_heads * 36 * hd; }

// places in a block's 9 HD words: of the word that holds a key code (token t of the block, channel), a value code, a group's parameters; and a code's first bit
TGX_KV4 int kv4_word(int i, int q, int r) { return ((i >> 2) * 64 + 16 * q + r) * 4 + (i & 3); }
TGX_KV4 int kv4_key_word(int hd, int t, int ch) { return kv4_word((t >> 4) * (hd / 32) + (ch >> 5), (ch >> 3) & 3, t & 15); }
TGX_KV4 int kv4_value_word(int hd, int t, int ch) { return 4 * hd + kv4_word(ch >> 4, (t & 15) >> 2, ch & 15); }
TGX_KV4 int kv4_param_word(int hd, int t, int value, int group) { return 8 * hd + (t * 2 + value) * (hd / 64) + group; }
TGX_KV4 int kv4_code_bit(int e) { return 4 * ((e >> 1) + 4 * (e & 1)); }
TGX_KV4 int kv4_key_bit(int ch) { return kv4_code_bit(ch & 7); }
TGX_KV4 int kv4_value_bit(int t) { return kv4_code_bit((t & 3) + 4 * ((t >> 4) & 1)); }
TGX_KV4 int kv4_value_token(int q, int e) { return e < 4 ? 4 * q + e : 12 + 4 * q + e; }      // the token of a value word's code e

// A scale enters as a positive factor of the scores and a sign of the queries (0: queries of zero), so that the largest score is the largest before the scale
inline void kv4_scale(Kv4Args& a, float scale) {
  a.q_sign = scale > 0.f ? 1.f : scale < 0.f ? -1.f : 0.f;
  a.scale_log2 = scale == 0.f ? 1.f : (scale < 0.f ? -scale : scale) * 1.4426950408889634f;
  a.gap = std::min(8.f / a.scale_log2, 1e30f);
}

// pages [lo, hi) that split `split` of `splits` walks for columns at positions first .. last
struct Kv4Range { int lo, hi; };
TGX_KV4 Kv4Range kv4_range(int first, int last, int window, int table_len, int split, int splits) {
  const int key_lo = window > 0 && first - window + 1 > 0 ? first - window + 1 : 0;
  const int lo = key_lo >> KV4_PAGE_SHIFT, all = last < 0 ? 0 : (last >> KV4_PAGE_SHIFT) + 1, hi = all < table_len ? all : table_len;
  const int per = hi > lo ? (hi - lo + splits - 1) / splits : 0;
  const long long p0 = lo + (long long)split * per, p1 = p0 + per;
  return Kv4Range{(int)(p0 < hi ? p0 : hi), (int)(p1 < hi ? p1 : hi)};
}

// How a batch's attention is divided: kw > 1 = the kw waves of a workgroup share nt * 16 columns (token, query head) and divide the keys, kw 1 = four waves divide the columns;
// tiles workgroups of columns, splits of the keys between workgroups (their records meet in a launch of their own)
struct Kv4Plan { int kw, nt, tiles, splits; };
inline Kv4Plan kv4_plan(int entries, int max_count, int kv_heads, int group, int hd, int window, long long max_keys, int num_cus) {
  Kv4Plan p;
  const long long cols = (long long)max_count * group;
  p.kw = cols <= 32 ? 4 : 1;
  p.nt = p.kw > 1 && cols <= 16 ? 1 : 2;
  const int per = 16 * p.nt * (p.kw > 1 ? 1 : 4);
  p.tiles = (int)((cols + per - 1) / per);
  const long long keys = window > 0 ? std::min<long long>(max_keys, (long long)window + max_count) : max_keys;
  const long long pages = std::max<long long>(1, (keys + KV4_PAGE - 1) / KV4_PAGE);
  const long long wgs = std::max<long long>(1, (long long)entries * kv_heads * p.tiles);
  // Two workgroups a compute unit where the waves divide the keys, one where they divide the columns: with more, a wave walks fewer blocks behind the same way in and out.  us, one / two / three / four
  // workgroups a compute unit, four waves each: 32 rows of up to 4096 tokens, head_dim 128, 33.3 / 24.7 / 30.0 / 32.5; one of 131071 45.1 / 33.8 / 33.4 / 39.1; 64 of 1500, head_dim 64,
  // 11.7 / 8.9 / 10.4 / 11.8.
  const long long want = ((p.kw > 1 ? 2ll : 1ll) * num_cus + wgs - 1) / wgs;
  p.splits = (int)std::max<long long>(1, std::min<long long>({want, pages, 256}));
  // The records' launch and the way to it cost 3.3 us; a page of 128 tokens walked by one workgroup 0.29 us at head_dim 64, 0.5 at 128 (eight waves).  us whole / split, eight heads of one row: head_dim 64,
  // 700 tokens 6.3 / 8.1, 1024 7.1 / 8.1, 1500 8.6 / 8.1; head_dim 128, 512 8.1 / 9.1, 700 8.8 / 9.2, 1024 10.5 / 9.3; 16 rows of head_dim 128, 1024 11.3 / 12.7, 2048 16.3 / 15.5.
  if (p.kw > 1 && pages * (p.splits - 1) * (hd / 64) <= 12ll * p.splits) p.splits = 1;
  // A single token's keys whole in a workgroup: eight waves where there is a compute unit for each workgroup (16 rows of head_dim 128, 2048 tokens, four waves / eight: 17.4 / 16.3;
  // one row of head_dim 64, 1024: 7.4 / 7.1) or the walk is long (64 rows of eight heads, head_dim 64: 1024 tokens 11.5 / 12.7, 3000 24.9 / 23.0)
  if (max_count == 1 && group <= 8 && p.splits == 1 && (wgs <= num_cus ? pages > 2 : pages >= 16)) p.kw = 8;
  return p;
}
inline size_t kv4_part_floats(const Kv4Plan& p, long long rows, int hd) { return p.splits > 1 ? (size_t)rows * p.splits * (hd + 2) : 0; }      // workspace of the splits' records

// A model's steps: the keys that the work of a step over `keys` of them is divided for (a power of two, part of a captured step's identity), and the workspace that the steps of up to
// max_batch rows (four positions of a prompt by steps) over up to max_ctx keys need
inline int kv4_bucket(long long keys) { int b = 256; while (b < keys && b < (1 << 30)) b *= 2; return b; }
inline size_t kv4_step_floats(int max_batch, int heads, int kv_heads, int hd, long long max_ctx, int num_cus) {
  size_t need = 0;
  for (int R = 1; R <= std::max(4, max_batch); R++)
    for (long long keys = kv4_bucket(1);; keys *= 2) {
      need = std::max(need, kv4_part_floats(kv4_plan(R, 1, kv_heads, heads / kv_heads, hd, 0, keys, num_cus), (long long)R * heads, hd));
      if (keys >= max_ctx) break;
    }
  return need;
}

}  // namespace tgx
