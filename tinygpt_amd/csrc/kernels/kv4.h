// kv4.h — a key / value cache held in 4 bits: the append that fills its pages, the read that gives the values back, attention over it, page copies.
//
// Format.  64 neighbouring channels of a token and head are a group: 16 levels lo + step n.
//   lo = bf16(min x, rounded down), step = max(bf16(f32((max x - lo) * (1 / 15)), rounded up), 2^-126), n = min(15, rint(f32(f32(x - lo) * f32(1 / step))))
// every operation one IEEE f32 operation, so that the codes follow from the inputs alone, whichever kernel writes them.  Rounding lo down and step up keeps
// every x inside the levels; x is off by half a step at most.  A group with a value that is not finite (or whose spread is not) is stored as lo = NaN, step = 0:
// its values read as NaN, they do not pass for numbers.  4.5 bits a channel; a group of 64 is one MFMA's 32 channels twice, so that a score's factors stay
// outside of the products (below).
//
// Layout.  A page holds KV_BLOCK = 128 tokens: [kv_heads][4 blocks of 32 tokens][36 HD bytes].  A block: key codes (16 HD bytes), value codes (16 HD), parameters
// (4 HD).  The codes lie in the order in which the matrix cores take them as operands, eight to a 32-bit word, so that a lane's 16-byte load is its operand and
// nothing passes through LDS: word (part * 64 + lane) * 4 + w, lane = 16 q + r, i = 4 part + w,
//   keys    token 16 (i / (HD / 32)) + r, channels 32 (i % (HD / 32)) + 8 q + e        (the A operand of a 16 x 16 x 32 product: rows tokens)
//   values  channel 16 i + r, token 4 q + e (e < 4) or 16 + 4 q + e - 4                 (the B operand, its contraction in the order in which the scores' lanes hold the tokens)
// e = 0 .. 7 at bit 4 (e / 2 + 4 (e % 2)).
// Parameters: [32 tokens][keys, values][HD / 64] words, lo in the low half, step in the high.
#pragma once
#include "common.h"
#include "../kv4_plan.h"

namespace tgx {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;

template <int HD> constexpr int kv4_block_words() { return 9 * HD; }
static_assert(KV4_PAGE == KV_BLOCK, "a page of the 4-bit cache holds as many tokens as one of the 16-bit cache");

__device__ __forceinline__ float kv4_load(const void* p, long long i, int dt) {
  if (dt == DT_F32) return static_cast<const float*>(p)[i];
  const unsigned short u = static_cast<const unsigned short*>(p)[i];
  return dt == DT_BF16 ? bf16_to_f32(u) : f16_bits_to_f32(u);
}
// ---- one group's levels ----------------------------------------------------------------------------------------------------------------------------
struct Kv4Levels { float lo, inv; unsigned int word; };       // word: the group's parameter word
__device__ __forceinline__ Kv4Levels kv4_levels(float mn, float mx, bool bad) {
  Kv4Levels g;
  const unsigned int lb = __float_as_uint(mn);
  g.lo = __uint_as_float((mn < 0.f ? lb + 0xffffu : lb) & 0xffff0000u);
  const float spread = __fsub_rn(mx, g.lo);
  const float step = fmaxf(__uint_as_float((__float_as_uint(__fmul_rn(spread, 1.0f / 15.0f)) + 0xffffu) & 0xffff0000u), 1.17549435e-38f);
  g.inv = __fdiv_rn(1.0f, step);
  if (bad || !(spread <= 3.402823466e38f)) { g.inv = 0.f; g.lo = 0.f; g.word = 0x00007fc0u; }      // codes 0, lo NaN, step 0
  else g.word = (__float_as_uint(g.lo) >> 16) | __float_as_uint(step);
  return g;
}
// a value that is not finite only meets a group that is stored as NaN: its codes are 0
__device__ __forceinline__ unsigned int kv4_code(float x, const Kv4Levels& g) {
  const float n = rintf(__fmul_rn(__fsub_rn(x, g.lo), g.inv));
  return n > 0.f ? (unsigned int)fminf(n, 15.f) : 0u;      // (a NaN is not above 0)
}
__device__ __forceinline__ bool kv4_not_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u; }

// minimum / maximum over 32 neighbouring lanes, every lane gets it
template <bool MAX> __device__ __forceinline__ float kv4_extreme32(float v) {
  auto f = [](float x, float y) { return MAX ? fmaxf(x, y) : fminf(x, y); };
  v = f(v, dpp_mov<0xB1, 0xf>(v));
  v = f(v, dpp_mov<0x4E, 0xf>(v));
  v = f(v, dpp_mov<0x141, 0xf>(v));
  v = f(v, dpp_mov<0x140, 0xf>(v));
  const u32x2 r = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// One token of one kv head by one wave: a lane takes two channels (HD 64: lanes 0-31 the key, 32-63 the value; HD 128: the key, then the value), a group is 32
// lanes.  A value word holds seven other tokens' codes, which stay: OWNED = nothing else writes the word in this launch, and it is read and stored; otherwise the
// eight codes of a word may come from several entries and the change goes in by an atomic exclusive or, whose result does not depend on the order.
template <int HD, bool OWNED>
__device__ __forceinline__ void kv4_append_one(const Kv4Args& a, unsigned int* page, int e, long long tok, int pos, int kvh) {
  constexpr int ROUNDS = HD / 64;
  const int lane = threadIdx.x & 63;
  const int t = pos & (KV4_BLK - 1);
  unsigned int* blk = page + (size_t)((pos >> 5) & 3) * kv4_block_words<HD>();
  float x[ROUNDS][2];
#pragma unroll
  for (int r = 0; r < ROUNDS; r++) {
    const bool val = HD == 64 ? lane >= 32 : r == 1;
    const int ch = HD == 64 ? 2 * (lane & 31) : 2 * lane;
    const long long at = kv4_kv_at(a, e, tok, pos, kvh, val) + ch;
    const void* src = val ? a.v : a.k;
    x[r][0] = kv4_load(src, at, a.kv_dt);
    x[r][1] = kv4_load(src, at + 1, a.kv_dt);
  }
#pragma unroll
  for (int r = 0; r < ROUNDS; r++) {
    const bool val = HD == 64 ? lane >= 32 : r == 1;
    const int ch = HD == 64 ? 2 * (lane & 31) : 2 * lane, g = ch >> 6;
    const float bad = kv4_extreme32<true>(kv4_not_finite(x[r][0]) || kv4_not_finite(x[r][1]) ? 1.f : 0.f);
    const Kv4Levels lv = kv4_levels(kv4_extreme32<false>(fminf(x[r][0], x[r][1])), kv4_extreme32<true>(fmaxf(x[r][0], x[r][1])), bad != 0.f);
    const unsigned int n0 = kv4_code(x[r][0], lv), n1 = kv4_code(x[r][1], lv);
    if ((lane & 31) == 0) blk[kv4_param_word(HD, t, val ? 1 : 0, g)] = lv.word;
    // a key word: eight channels = four lanes
    const int i4 = 4 * (lane & 3);
    int kw = (int)((n0 << i4) | (n1 << (i4 + 16)));
    kw |= __builtin_amdgcn_update_dpp(0, kw, 0xB1, 0xf, 0xf, false);
    kw |= __builtin_amdgcn_update_dpp(0, kw, 0x4E, 0xf, 0xf, false);
    if (!val) {
      if ((lane & 3) == 0) blk[kv4_key_word(HD, t, ch)] = (unsigned int)kw;
    } else {
      const int bit = kv4_value_bit(t);
#pragma unroll
      for (int c = 0; c < 2; c++) {
        unsigned int* w = blk + kv4_value_word(HD, t, ch + c);
        const unsigned int n = (c ? n1 : n0) << bit, m = 15u << bit;
        if constexpr (OWNED) *w = (*w & ~m) | n;
        else {
          const unsigned int old = __hip_atomic_load(w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          __hip_atomic_fetch_xor(w, (old ^ n) & m, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
      }
    }
  }
}

// Few tokens: a wave a (entry, token, kv head).
template <int HD>
__global__ __launch_bounds__(64) void kv4_append_token_kernel(const Kv4Args a) {
  const Kv4Entry en = kv4_entry(a, blockIdx.z);
  const int i = blockIdx.y, pos = en.start + i;
  if (i >= en.count || pos < 0) return;
  unsigned int* page = kv4_page(a, en.seq, pos >> KV4_PAGE_SHIFT, blockIdx.x, HD);
  if (page) kv4_append_one<HD, false>(a, page, blockIdx.z, en.tok0 + i, pos, blockIdx.x);
}

// Portions: a workgroup of 2 HD threads a (entry, block of 32 positions, kv head).  Two neighbouring lanes take a group of one token, 32 channels each (32 tokens x HD / 64 groups x {key, value}):
// one exchange between them gives the levels.  The values' codes pass through LDS as bytes [token][channel], where a value word finds its eight tokens.  Bound by memory where there is
// enough of it (16 rows of 2048 tokens, eight heads of 128: 34 us, 4.9 TB/s) and by the way through one block where there is not (4.8 us; a lane a whole group 10.5).
template <int HD, int DT>
__global__ __launch_bounds__(2 * HD) void kv4_append_block_kernel(const Kv4Args a) {
  constexpr int G = HD / 64, LS = HD + 4;                      // bytes of a token in LDS
  __shared__ __attribute__((aligned(16))) unsigned char s[KV4_BLK * LS];
  const Kv4Entry en = kv4_entry(a, blockIdx.z);
  const int kvh = blockIdx.x, tid = threadIdx.x;
  if (en.count < 1) return;
  const int s0 = max(en.start, 0), b = (s0 >> 5) + blockIdx.y;      // block of positions
  const int p0 = max(s0, b * KV4_BLK), p1 = min(en.start + en.count, (b + 1) * KV4_BLK);
  if (p0 >= p1) return;
  unsigned int* page = kv4_page(a, en.seq, b >> 2, kvh, HD);
  if (!page) return;
  unsigned int* blk = page + (size_t)(b & 3) * kv4_block_words<HD>();
  {
    const int half = tid & 1, item = tid >> 1, val = item / (32 * G), rest = item % (32 * G), t = rest / G, g = rest % G, pos = b * KV4_BLK + t;
    const bool in = pos >= p0 && pos < p1;
    const int sp = in ? pos : p0;                               // (a lane without a token reads one that is there)
    const long long tok = en.tok0 + sp - en.start;
    const elem_t<DT>* src = static_cast<const elem_t<DT>*>(val ? a.v : a.k) + kv4_kv_at(a, blockIdx.z, tok, sp, kvh, val) + g * 64 + 32 * half;
    float x[32];
    if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
#pragma unroll
      for (int i = 0; i < 4; i++) slice_unpack<DT>(load_slice<DT>(src, i), x + 8 * i);
    } else {
#pragma unroll
      for (int i = 0; i < 32; i++) x[i] = elem_to_f32<DT>(src[i]);
    }
    float mn = x[0], mx = x[0];
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 32; i++) { mn = fminf(mn, x[i]); mx = fmaxf(mx, x[i]); bad |= kv4_not_finite(x[i]); }
    mn = fminf(mn, dpp_mov<0xB1, 0xf>(mn));
    mx = fmaxf(mx, dpp_mov<0xB1, 0xf>(mx));
    const float wrong = bad ? 1.f : 0.f;
    const Kv4Levels lv = kv4_levels(mn, mx, fmaxf(wrong, dpp_mov<0xB1, 0xf>(wrong)) != 0.f);
    if (in && half == 0) blk[kv4_param_word(HD, t, val, g)] = lv.word;
    if (!val) {
#pragma unroll
      for (int q = 0; q < 4; q++) {
        unsigned int w = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) w |= kv4_code(x[8 * q + e], lv) << kv4_code_bit(e);
        if (in) blk[kv4_key_word(HD, t, 64 * g + 32 * half + 8 * q)] = w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) {
        unsigned int w = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) w |= kv4_code(x[4 * i + e], lv) << (8 * e);
        *reinterpret_cast<unsigned int*>(s + t * LS + g * 64 + 32 * half + 4 * i) = w;
      }
    }
  }
  __syncthreads();
  // value words: a thread takes two neighbouring channels of a quarter's eight tokens
  const int q = tid / (HD / 2), c2 = 2 * (tid % (HD / 2));
  unsigned int w[2] = {0, 0}, m = 0;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const int t = kv4_value_token(q, e), pos = b * KV4_BLK + t, bit = kv4_code_bit(e);
    const unsigned int cs = *reinterpret_cast<const unsigned short*>(s + t * LS + c2);
    if (pos >= p0 && pos < p1) {
      m |= 15u << bit;
      w[0] |= (cs & 15u) << bit;
      w[1] |= ((cs >> 8) & 15u) << bit;
    }
  }
#pragma unroll
  for (int c = 0; c < 2; c++) {
    unsigned int* dst = blk + kv4_value_word(HD, 4 * q, c2 + c);
    if (m == 0xffffffffu) *dst = w[c];
    else if (m) {
      const unsigned int old = __hip_atomic_load(dst, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_fetch_xor(dst, (old ^ w[c]) & m, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
}

// The values that the pages hold for the batch's tokens: a wave a (entry, block of 32 positions, kv head).  Bound by its stores, 16 bits or more for 4.5 that it reads: four rows of up to 4096
// tokens, eight heads of 128, 14.4 us (4.0 TB/s); a token of each of 64 rows 3.9 us.
template <int HD, int DT>
__global__ __launch_bounds__(64) void kv4_read_kernel(const Kv4Args a) {
  constexpr int PARTS = HD / 64;
  __shared__ __attribute__((aligned(16))) unsigned char s[KV4_BLK * (HD + 8)];      // (eight bytes at a time below)
  const Kv4Entry en = kv4_entry(a, blockIdx.z);
  const int kvh = blockIdx.x, lane = threadIdx.x, q = lane >> 4, r = lane & 15;
  if (en.count < 1) return;
  const int s0 = max(en.start, 0), b = (s0 >> 5) + blockIdx.y;
  const int p0 = max(s0, b * KV4_BLK), p1 = min(en.start + en.count, (b + 1) * KV4_BLK);
  if (p0 >= p1) return;
  const unsigned int* page = kv4_page(a, en.seq, b >> 2, kvh, HD);
  elem_t<DT>* ko = static_cast<elem_t<DT>*>(a.k);
  elem_t<DT>* vo = static_cast<elem_t<DT>*>(a.v);
  if (!page) {      // tokens without a page read as zeros
    for (int p = p0; p < p1; p++)
      for (int c = lane; c < HD; c += 64) {
        const long long tok = en.tok0 + p - en.start;
        ko[tok * a.k_ts + kvh * a.k_hs + c] = 0;
        vo[tok * a.v_ts + kvh * a.v_hs + c] = 0;
      }
    return;
  }
  const unsigned int* blk = page + (size_t)(b & 3) * kv4_block_words<HD>();
#pragma unroll
  for (int p = 0; p < PARTS; p++) {
    const u32x4 w = reinterpret_cast<const u32x4*>(blk)[p * 64 + lane], vw = reinterpret_cast<const u32x4*>(blk + 4 * HD)[p * 64 + lane];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int i = 4 * p + j, t = 16 * (i / (HD / 32)) + r, chunk = i % (HD / 32), pos = b * KV4_BLK + t;
      if (pos >= p0 && pos < p1) {
        const unsigned int par = blk[kv4_param_word(HD, t, 0, chunk >> 1)];
        const float lo = bf16_lo(par), st = bf16_hi(par);
        elem_t<DT>* dst = ko + (en.tok0 + pos - en.start) * a.k_ts + kvh * a.k_hs + 32 * chunk + 8 * q;
#pragma unroll
        for (int e = 0; e < 8; e++) dst[e] = f32_to_elem<DT>(fmaf(st, (float)((w[j] >> kv4_code_bit(e)) & 15u), lo));
      }
#pragma unroll
      for (int e = 0; e < 8; e++) s[kv4_value_token(q, e) * (HD + 8) + 16 * i + r] = (unsigned char)((vw[j] >> kv4_code_bit(e)) & 15u);
    }
  }
  __syncthreads();
  for (int item = lane; item < KV4_BLK * HD / 8; item += 64) {
    const int t = item / (HD / 8), c8 = item % (HD / 8), pos = b * KV4_BLK + t;
    if (pos < p0 || pos >= p1) continue;
    const unsigned int par = blk[kv4_param_word(HD, t, 1, c8 >> 3)];
    const float lo = bf16_lo(par), st = bf16_hi(par);
    elem_t<DT>* dst = vo + (en.tok0 + pos - en.start) * a.v_ts + kvh * a.v_hs + 8 * c8;
    const u32x2 cs = *reinterpret_cast<const u32x2*>(s + t * (HD + 8) + 8 * c8);
#pragma unroll
    for (int e = 0; e < 8; e++) dst[e] = f32_to_elem<DT>(fmaf(st, (float)((cs[e >> 2] >> (8 * (e & 3))) & 255u), lo));
  }
}

// ---- attention ------------------------------------------------------------------------------------------------------------------------------------------
// S^T = K Q^T with the codes as the operand: a score is sum_g step_g (q_g . n_g) + lo_g sum(q_g), so that a product of 16 tokens x 16 query columns (column = token of the
// entry, query head of the kv head) costs two fused multiply-adds a score and group and no value is worked out.  O = P V the same way: the weights p step_g (bf16, TP terms of
// them) meet the codes, the lo part is summed in f32.  Lane (q, r) holds the scores of column r, tokens 4 q .. 4 q + 3 of a 16-token tile: as it needs them as the A
// operand of P V, whose contraction runs over the tokens in the order of the value words.
// QT: a query's and an output's type.  TQ, TP: 16-bit terms of a query and of a weight.  Queries in bf16 are one term exactly, in fp16 two, in fp32 three (2^-25).  Of a weight, two (2^-17)
// leave an output in 16 bits what its own rounding leaves, three one in 32.  A model's steps take its 32-bit activations as two terms (2^-17), as its products do.  (One, as coarse as an output in bf16, with the values about
// the middle of their levels: portions in 15 % less time, one long row in 8 %, and outputs 1.4 times as far from 64 bits.)
// A word's codes as bf16 numbers, exactly: a byte n of 0 .. 15 is the fp8 (e4m3) number n / 512, and the conversion scales.  They come in the order e = 0, 4, 1, 5, 2, 6, 3, 7, in which
// what they are multiplied with is laid out (kv4_slot: the code at a place).
__device__ __forceinline__ bf16x8_t kv4_frag(unsigned int w) {
  const unsigned int a = w & 0x0f0f0f0fu, b = (w >> 4) & 0x0f0f0f0fu;
  u32x4 f;
  f[0] = __builtin_bit_cast(unsigned int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 512.f, false));
  f[1] = __builtin_bit_cast(unsigned int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 512.f, true));
  f[2] = __builtin_bit_cast(unsigned int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 512.f, false));
  f[3] = __builtin_bit_cast(unsigned int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 512.f, true));
  return __builtin_bit_cast(bf16x8_t, f);
}
constexpr int kv4_slot[8] = {0, 4, 1, 5, 2, 6, 3, 7};
// 32-bit outputs (TP 3) take the values' codes and levels about their middle, step (n - 7.5) and lo + 7.5 step: values of both signs leave a sum far below that of their codes, whose
// roundings would stay in it.  And a step's products are summed from zero and join the sums in f32: the matrix unit cuts off what lies below its largest term's last bits.  A window
// of 4096 keys: 1.8e-6 from the 64-bit sums and 21.8 us without either, 5e-7 and 23.8 us so (plain 32-bit sums of the values: 8e-7); the keys' codes about their middle too, 3e-7 and 25.7 us.
template <int TP> constexpr bool kv4_about_middle() { return TP == 3; }
template <int TP> __device__ __forceinline__ bf16x8_t kv4_operand(unsigned int w) {
  if constexpr (!kv4_about_middle<TP>()) return kv4_frag(w);
  // a byte of sign and |2 n - 15| is the fp8 number (2 n - 15) / 512; codes below 8 turn round
  auto centred = [](unsigned int n) {
    const unsigned int low = ~n & 0x08080808u;
    return (((n ^ (low - (low >> 3))) & 0x07070707u) << 1) | 0x01010101u | (low << 4);
  };
  const unsigned int a = centred(w & 0x0f0f0f0fu), b = centred((w >> 4) & 0x0f0f0f0fu);
  u32x4 f;
  f[0] = __builtin_bit_cast(unsigned int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 256.f, false));
  f[1] = __builtin_bit_cast(unsigned int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 256.f, true));
  f[2] = __builtin_bit_cast(unsigned int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 256.f, false));
  f[3] = __builtin_bit_cast(unsigned int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 256.f, true));
  return __builtin_bit_cast(bf16x8_t, f);
}
// Outputs in 16 bits (TP 2) keep the codes as they are, and a walk's products stay in the matrix unit's sums.  Those are of one sign and grow with the keys while the values' own sum does not: a
// sum's roundings, 2^-24 of it each, come to more than an output's own rounding over some 10^4 keys (1024 tokens in fp16 behind 32768: 4.4e-4 from 64 bits, behind 131072 1.6e-3; the rounding
// 2.1e-4).  So the part of the los, of the other sign, joins them every KV4_FOLD blocks, which leaves the values' sum:
// 8e-6 of a row beside its output's rounding at any length, which is what two terms of a weight leave, for 2 % of a portion's time (476 us: 486) and 1 of one long row's.
constexpr int KV4_FOLD = 16;
template <int TP> __device__ __forceinline__ float kv4_base(float lo, float step) { return kv4_about_middle<TP>() ? fmaf(7.5f, step, lo) : lo; }
// over the lanes of equal r: lanes 16 and 32 further swap in the vector registers
__device__ __forceinline__ float kv4_max_quarters(float v) {
  u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  v = fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1]));
  w = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  return fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1]));
}
__device__ __forceinline__ float kv4_sum_quarters(float v) {
  u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  v = __uint_as_float(w[0]) + __uint_as_float(w[1]);
  w = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  return __uint_as_float(w[0]) + __uint_as_float(w[1]);
}
// what weights of an old reference (a score) are of a new one.  Weights are 2^(score scale - reference scale) with the second product rounded: the factor is made of the rounded ones, or
// sums of different references would be off by their difference.  Records of sums hold the rounded product.
__device__ __forceinline__ float kv4_factor(float was, float is, float scale) {
#pragma clang fp contract(off)
  const float a = was * scale, b = is * scale;
  return __builtin_amdgcn_exp2f(a - b);
}
// the page of a block, -1: none.  Tables are read through the scalar cache: an entry in front of its use costs no vector register and waits for no vector load
__device__ __forceinline__ int kv4_page_id(const Kv4Args& a, int seq, int b, int b_hi) {
  if (b >= b_hi || (b >> 2) >= a.table_len) return -1;
  const int* at = a.table + (long long)seq * a.table_stride + (b >> 2);
  const int p = *(const __attribute__((address_space(4))) int*)at;
  return p >= 0 && p < a.pages ? p : -1;
}
// eight neighbouring channels of a row
template <int DT>
__device__ __forceinline__ void kv4_load8(const void* p, long long i, float x[8]) {
  const elem_t<DT>* e = static_cast<const elem_t<DT>*>(p) + i;
  if ((reinterpret_cast<uintptr_t>(e) & 15) == 0) slice_unpack<DT>(load_slice<DT>(e, 0), x);
  else {
#pragma unroll
    for (int c = 0; c < 8; c++) x[c] = elem_to_f32<DT>(e[c]);
  }
}
// four neighbouring channels of an output; mode: rounded to a storage type first (32-bit outputs; option act.round16 of a model)
template <int DT>
__device__ __forceinline__ void kv4_store4(void* p, long long i, const f32x4 v, int mode) {
  elem_t<DT>* e = static_cast<elem_t<DT>*>(p) + i;
  if constexpr (DT == DT_F32) {
    f32x4 r = v;
    if (mode) {
#pragma unroll
      for (int c = 0; c < 4; c++) r[c] = round_storage_mode(v[c], mode);
    }
    if ((reinterpret_cast<uintptr_t>(e) & 15) == 0) *reinterpret_cast<f32x4*>(e) = r;
    else {
#pragma unroll
      for (int c = 0; c < 4; c++) e[c] = r[c];
    }
  } else {
    elem_t<DT> h[4];
#pragma unroll
    for (int c = 0; c < 4; c++) h[c] = f32_to_elem<DT>(v[c]);
    if ((reinterpret_cast<uintptr_t>(e) & 7) == 0) *reinterpret_cast<u32x2*>(e) = u32x2{h[0] | ((unsigned int)h[1] << 16), h[2] | ((unsigned int)h[3] << 16)};
    else {
#pragma unroll
      for (int c = 0; c < 4; c++) e[c] = h[c];
    }
  }
}
template <int DT>
__device__ __forceinline__ void kv4_store1(void* p, long long i, float v, int mode) {
  static_cast<elem_t<DT>*>(p)[i] = f32_to_elem<DT>(DT == DT_F32 && mode ? round_storage_mode(v, mode) : v);
}

// a block's codes and parameters on their way: key and value words as operands, the parameters of token (lane & 31)
template <int HD> struct Kv4Raw {
  u32x4 k[HD / 64], v[HD / 64];
  unsigned int p[HD / 32];
  __device__ __forceinline__ void load(const unsigned int* blk, int lane) {
#pragma unroll
    for (int i = 0; i < HD / 64; i++) k[i] = load_nt(reinterpret_cast<const u32x4*>(blk) + i * 64 + lane);
    if constexpr (HD == 128) { const u32x4 w = load_nt(reinterpret_cast<const u32x4*>(blk + 8 * HD) + (lane & 31)); p[0] = w[0]; p[1] = w[1]; p[2] = w[2]; p[3] = w[3]; }
    else { const u32x2 w = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(blk + 8 * HD) + (lane & 31)); p[0] = w[0]; p[1] = w[1]; }
#pragma unroll
    for (int i = 0; i < HD / 64; i++) v[i] = load_nt(reinterpret_cast<const u32x4*>(blk + 4 * HD) + i * 64 + lane);
  }
};

// The sums of NT tiles of 16 query columns over the blocks that a wave walks.
template <int HD, int NT, int QT, int TQ, int TP>
struct Kv4Sums {
  static constexpr int G = HD / 64, CH = HD / 32, CT = HD / 16;
  bf16x8_t qf[NT][CH][TQ];
  // The sums of a query's channels of a group, which meet the los: in f32, or for queries of one term (whose operands leave the registers) as three terms (2^-25) of a product of its own, at
  // places 3 g .. 3 g + 2 of quarter 0
  static constexpr bool LO_PRODUCT = TQ == 1;
  float qsum[NT][LO_PRODUCT ? 1 : G];
  bf16x8_t qlo[LO_PRODUCT ? NT : 1];
  int pos[NT];                                                // a column's position; -1: no column
  f32x4 o[NT][CT];
  float m[NT], l[NT], lov[NT][G];                             // m: the reference of the weights, in scores before the scale (records hold it behind it)

  __device__ __forceinline__ void start(const Kv4Args& a, const Kv4Entry& en, int kvh, int col0, int ncol, int q4, int r16) {
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const int c = col0 + 16 * t + r16, cc = min(c, ncol - 1), i = en.count == 1 ? 0 : cc / a.group, h = kvh * a.group + cc - i * a.group;
      pos[t] = c < ncol ? en.start + i : -1;
      const long long base = (en.tok0 + i) * a.q_ts + h * a.q_hs + 8 * q4;
      m[t] = -INFINITY; l[t] = 0.f;
#pragma unroll
      for (int g = 0; g < G; g++) lov[t][g] = 0.f;
      float sum[G] = {};
#pragma unroll
      for (int x = 0; x < CT; x++) o[t][x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ch = 0; ch < CH; ch++) {
        float x[8];
        kv4_load8<QT>(a.q, base + 32 * ch, x);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] *= a.q_sign;
#pragma unroll
        for (int term = 0; term < TQ; term++) {
          u32x4 f;
#pragma unroll
          for (int e = 0; e < 4; e++) {
            f[e] = pack_bf16(x[kv4_slot[2 * e]], x[kv4_slot[2 * e + 1]]);
            sum[ch / 2] += bf16_lo(f[e]) + bf16_hi(f[e]);
            x[kv4_slot[2 * e]] -= bf16_lo(f[e]); x[kv4_slot[2 * e + 1]] -= bf16_hi(f[e]);
          }
          qf[t][ch][term] = __builtin_bit_cast(bf16x8_t, f);
        }
      }
#pragma unroll
      for (int g = 0; g < G; g++) sum[g] = kv4_sum_quarters(sum[g]);
      if constexpr (LO_PRODUCT) {
        u32x4 f = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
        for (int g = 0; g < G; g++)
#pragma unroll
          for (int i = 3 * g; i < 3 * g + 3; i++) {
            const unsigned int term = pack_bf16(sum[g], 0.f) & 0xffffu;
            sum[g] -= bf16_lo(term);
            f[i >> 1] |= q4 == 0 ? term << (16 * (i & 1)) : 0u;
          }
        qlo[t] = __builtin_bit_cast(bf16x8_t, f);
      } else {
#pragma unroll
        for (int g = 0; g < G; g++) qsum[t][g] = sum[g];
      }
    }
  }

  // the part of the los joins o
  __device__ __forceinline__ void fold(int q4) {
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int g = 0; g < G; g++) {
        const float lg = kv4_sum_quarters(lov[t][g]);
        lov[t][g] = 0.f;
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const float add = __shfl(lg, 4 * q4 + r, 64);
#pragma unroll
          for (int c = 0; c < 4; c++) o[t][4 * g + c][r] += add;
        }
      }
  }

  // One block of 32 tokens from position t0 on.  sp: the wave's LDS for the parameters, which every lane needs of the four tokens of its scores.  MASK: some column does not
  // see some token of the block; what is not seen is selected away, whatever it holds.  In phases that the compiler does not mix: mixed, their registers are half again as many.
  // key, value: the block's operands, by their number.
  template <bool MASK, typename Keys, typename Values>
  __device__ __forceinline__ void block(const Keys& key, const Values& value, const unsigned int (&par)[HD / 32], int t0, int window, float scale, float gap, float* sp, int lane) {
    const int q4 = lane >> 4;
    // Each token's levels become numbers once: floats [step of the keys' groups, lo of them, step of the values', base of them][32 tokens]; lanes of 32 and beyond take the values'
    {
      const bool values = lane >= 32;
#pragma unroll
      for (int g = 0; g < G; g++) {
        const unsigned int w = values ? par[G + g] : par[g];
        const float st = bf16_hi(w), lo = bf16_lo(w);
        float* to = sp + (values ? 64 * G : 0) + (lane & 31);
        to[32 * g] = st;
        to[32 * (G + g)] = values ? kv4_base<TP>(lo, st) : lo;
      }
    }
    wave_fence();
    // the steps and los (bases) of a lane's four tokens of tile i: keys (0) or values (1)
    auto levels = [&](int which, int i, int g, f32x4& st, f32x4& lo) {
      st = *reinterpret_cast<const f32x4*>(sp + (which * 2 * G + g) * 32 + 16 * i + 4 * q4);
      lo = *reinterpret_cast<const f32x4*>(sp + (which * 2 * G + G + g) * 32 + 16 * i + 4 * q4);
    };
    // the los of tile i's tokens as a row's operand: a token's lo at its group's three places, the same in every quarter (a product with zeros keeps a token's NaN to the token)
    bf16x8_t lof[2];
    if constexpr (LO_PRODUCT) {
      u32x2 w[G];
#pragma unroll
      for (int g = 0; g < G; g++) w[g] = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(par[g], par[g], false, false));
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const unsigned int a = __builtin_amdgcn_perm(w[0][i], w[0][i], 0x01000100u), b = __builtin_amdgcn_perm(w[G - 1][i], w[0][i], 0x05040100u);
        const unsigned int c = __builtin_amdgcn_perm(w[G - 1][i], w[G - 1][i], 0x01000100u);
        lof[i] = __builtin_bit_cast(bf16x8_t, u32x4{a, b, c, c});
      }
    }
    f32x4 sc[NT][2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (LO_PRODUCT) {
#pragma unroll
        for (int t = 0; t < NT; t++) sc[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lof[i], qlo[t], f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
      }
#pragma unroll
      for (int g = 0; g < G; g++) {
        bf16x8_t kf[2];
#pragma unroll
        for (int c = 0; c < 2; c++) kf[c] = key(i * CH + 2 * g + c);
        f32x4 st, z;
        levels(0, i, g, st, z);
#pragma unroll
        for (int t = 0; t < NT; t++) {
          f32x4 d = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < 2; c++)
#pragma unroll
            for (int term = 0; term < TQ; term++) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[c], qf[t][2 * g + c][term], d, 0, 0, 0);
#pragma unroll
          for (int r = 0; r < 4; r++) sc[t][i][r] = fmaf(st[r], d[r], LO_PRODUCT ? sc[t][i][r] : g == 0 ? z[r] * qsum[t][g] : fmaf(z[r], qsum[t][g], sc[t][i][r]));
        }
      }
    }
    float p[NT][2][4];
    bool seen[NT][2][4];
#pragma unroll
    for (int t = 0; t < NT; t++) {
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int j = t0 + 16 * i + 4 * q4 + r;
          seen[t][i][r] = !MASK || (j <= pos[t] && (window <= 0 || j > pos[t] - window));
          if (MASK && !seen[t][i][r]) sc[t][i][r] = -INFINITY;
          mx = fmaxf(mx, sc[t][i][r]);
        }
      mx = kv4_max_quarters(mx);
      // the sums keep their reference until a maximum passes it by 8 in the exponent (weights up to 256 then): few blocks rescale
      if (__any(mx > m[t] + gap)) {
        const float nm = fmaxf(m[t], mx), f = nm > m[t] ? kv4_factor(m[t], nm, scale) : 1.f;
        m[t] = nm;
        l[t] *= f;
#pragma unroll
        for (int g = 0; g < G; g++) lov[t][g] *= f;
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const float fr = __shfl(f, 4 * q4 + r, 64);
#pragma unroll
          for (int c = 0; c < CT; c++) o[t][c][r] *= fr;
        }
      }
      const float ref = -m[t] * scale;
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          p[t][i][r] = __builtin_amdgcn_exp2f(fmaf(sc[t][i][r], scale, ref));
          if (MASK && !seen[t][i][r]) p[t][i][r] = 0.f;
          l[t] += p[t][i][r];
        }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int g = 0; g < G; g++) {
      f32x4 vst[2], vlo[2];
#pragma unroll
      for (int i = 0; i < 2; i++) levels(1, i, g, vst[i], vlo[i]);
      u32x4 pf[NT][TP];
#pragma unroll
      for (int t = 0; t < NT; t++) {
        float ps[8];
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
          for (int r = 0; r < 4; r++) {
            ps[4 * i + r] = MASK && !seen[t][i][r] ? 0.f : p[t][i][r] * vst[i][r];
            lov[t][g] = MASK && !seen[t][i][r] ? lov[t][g] : fmaf(p[t][i][r], vlo[i][r], lov[t][g]);
          }
#pragma unroll
        for (int term = 0; term < TP; term++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            pf[t][term][e] = pack_bf16(ps[kv4_slot[2 * e]], ps[kv4_slot[2 * e + 1]]);
            if (term + 1 < TP) { ps[kv4_slot[2 * e]] -= bf16_lo(pf[t][term][e]); ps[kv4_slot[2 * e + 1]] -= bf16_hi(pf[t][term][e]); }
          }
      }
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const int x = 4 * g + c;
        const bf16x8_t vf = value(x);
#pragma unroll
        for (int t = 0; t < NT; t++) {
          f32x4 sum = kv4_about_middle<TP>() ? f32x4{0.f, 0.f, 0.f, 0.f} : o[t][x];
#pragma unroll
          for (int term = TP - 1; term >= 0; term--) sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, pf[t][term]), vf, sum, 0, 0, 0);
          if constexpr (kv4_about_middle<TP>()) o[t][x] += sum;
          else o[t][x] = sum;
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    wave_fence();
  }

  // The blocks b0, b0 + STEP, .. below b1, every one (MASK false) or only those of them outside of [skip0, skip1) (MASK true): one on its way while one is worked on, the page of the one behind on its way
  // before that.  A walk takes one kind of block: with both in one loop the compiler keeps two sets of sums.
  template <bool MASK, int STEP>
  __device__ __forceinline__ void walk(const Kv4Args& a, int seq, int kvh, int b0, int b1, int skip0, int skip1, float* sp, int lane) {
    const unsigned int* heads = a.pool + (size_t)kvh * (36 * HD);
    const size_t page_words = (size_t)a.kv_heads * (36 * HD);
    auto past = [&](int b) { return MASK && b >= skip0 && b < skip1 ? b + (skip1 - b + STEP - 1) / STEP * STEP : b; };
    Kv4Raw<HD> raw, nxt;
    int b = past(b0), bn = past(b + STEP), id = kv4_page_id(a, seq, b, b1), idn = kv4_page_id(a, seq, bn, b1);
    int walked = 0;
    if (id >= 0) raw.load(heads + id * page_words + (size_t)(b & 3) * kv4_block_words<HD>(), lane);
    while (b < b1) {
      const int bm = past(bn + STEP), idm = kv4_page_id(a, seq, bm, b1);
      if (idn >= 0) nxt.load(heads + idn * page_words + (size_t)(bn & 3) * kv4_block_words<HD>(), lane);
      if (id >= 0)
        block<MASK>([&](int x) { return kv4_frag(raw.k[x >> 2][x & 3]); }, [&](int x) { return kv4_operand<TP>(raw.v[x >> 2][x & 3]); }, raw.p, b * KV4_BLK, a.window, a.scale_log2, a.gap, sp, lane);
      if (!kv4_about_middle<TP>() && ++walked % KV4_FOLD == 0) fold(lane >> 4);
      raw = nxt; b = bn; id = idn; bn = bm; idn = idm;
    }
  }
  // the blocks [w0, w1) that columns at positions p0 .. p1 all see whole: t0 + 31 <= p0 and t0 > p1 - window
  static __device__ __forceinline__ void whole(const Kv4Args& a, int b_hi, int p0, int p1, int& w0, int& w1) {
    w1 = min(max((p0 + 1) >> 5, 0), b_hi);
    w0 = min(a.window > 0 && p1 - a.window + 1 > 0 ? (p1 - a.window + KV4_BLK) >> 5 : 0, w1);
  }
  // a wave's blocks (b_lo + first, in steps) of columns at positions p0 .. p1: those that every column sees whole, then the others
  template <int STEP>
  __device__ __forceinline__ void all(const Kv4Args& a, int seq, int kvh, int first_block, int b_hi, int p0, int p1, float* sp, int lane) {
    int w0, w1;
    whole(a, b_hi, p0, p1, w0, w1);
    int f = first_block;
    if (f < w0) f += (w0 - f + STEP - 1) / STEP * STEP;
    walk<false, STEP>(a, seq, kvh, f, w1, 0, 0, sp, lane);
    walk<true, STEP>(a, seq, kvh, first_block, b_hi, w0, w1, sp, lane);
  }

  // A workgroup's walk, four waves on the same blocks: a wave makes a quarter of a block's operands, all read them from LDS ([2][key operands, value operands][64] of them), which takes
  // three quarters of the conversions away.  Every wave comes here with the same blocks; mine: this wave has columns that see something up to position `until`.
  template <bool MASK>
  __device__ __forceinline__ void walk_shared(const Kv4Args& a, int seq, int kvh, int b0, int b1, int skip0, int skip1, bool mine, int until, bf16x8_t* so, float* sp, int wv, int lane) {
    constexpr int P = HD / 64, ONE = 2 * CT * 64;              // operands of a wave and kind, of a block
    const unsigned int* heads = a.pool + (size_t)kvh * (36 * HD);
    const size_t page_words = (size_t)a.kv_heads * (36 * HD);
    auto past = [&](int b) { return MASK && b >= skip0 && b < skip1 ? skip1 : b; };
    unsigned int k[P] = {}, v[P] = {}, par[HD / 32] = {}, par_next[HD / 32] = {};
    auto load = [&](int id, int b) {
      const unsigned int* blk = heads + id * page_words + (size_t)(b & 3) * kv4_block_words<HD>();
      const int x = wv * P, at = ((x >> 2) * 64 + lane) * 4 + (x & 3);
      if constexpr (P == 2) {
        const u32x2 kk = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(blk + at)), vv = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(blk + 4 * HD + at));
        k[0] = kk[0]; k[1] = kk[1]; v[0] = vv[0]; v[1] = vv[1];
        const u32x4 w = load_nt(reinterpret_cast<const u32x4*>(blk + 8 * HD) + (lane & 31));
        par_next[0] = w[0]; par_next[1] = w[1]; par_next[2] = w[2]; par_next[3] = w[3];
      } else {
        k[0] = __builtin_nontemporal_load(blk + at); v[0] = __builtin_nontemporal_load(blk + 4 * HD + at);
        const u32x2 w = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(blk + 8 * HD) + (lane & 31));
        par_next[0] = w[0]; par_next[1] = w[1];
      }
    };
    auto make = [&](bf16x8_t* to) {
#pragma unroll
      for (int i = 0; i < P; i++) { to[(wv * P + i) * 64 + lane] = kv4_frag(k[i]); to[(CT + wv * P + i) * 64 + lane] = kv4_operand<TP>(v[i]); }
#pragma unroll
      for (int i = 0; i < HD / 32; i++) par[i] = par_next[i];
    };
    int b = past(b0), id = kv4_page_id(a, seq, b, b1), cur = 0, walked = 0;
    if (b >= b1) return;
    if (id >= 0) { load(id, b); make(so); }
    int bn = past(b + 1), idn = kv4_page_id(a, seq, bn, b1);
    if (idn >= 0) load(idn, bn);
    __syncthreads();
    while (b < b1) {
      const int bm = past(bn + 1), idm = kv4_page_id(a, seq, bm, b1);
      const bf16x8_t* from = so + cur * ONE + lane;
      if (id >= 0 && mine && (!MASK || b * KV4_BLK <= until))
        block<MASK>([&](int x) { return from[x * 64]; }, [&](int x) { return from[(CT + x) * 64]; }, par, b * KV4_BLK, a.window, a.scale_log2, a.gap, sp, lane);
      if (!kv4_about_middle<TP>() && ++walked % KV4_FOLD == 0) fold(lane >> 4);
      cur ^= 1;
      if (idn >= 0) make(so + cur * ONE);
      if (idm >= 0) load(idm, bm);
      __syncthreads();
      b = bn; id = idn; bn = bm; idn = idm;
    }
  }

  // o becomes the columns' sums, l their denominators (over the four quarters)
  __device__ __forceinline__ void finish(int q4) {
    fold(q4);
#pragma unroll
    for (int t = 0; t < NT; t++) l[t] = kv4_sum_quarters(l[t]);
  }
};

// The waves' sums of up to 16 columns meet in LDS: so [KW][columns][HD], a thread takes four channels of a column through all waves; the split's record, or the output.
template <int HD, int KW, int DT>
__device__ __forceinline__ void kv4_meet(const Kv4Args& a, const Kv4Entry& en, int kvh, int split, int c0, int nv, const float* so, const float (*s_ml)[16][2]) {
  for (int item = threadIdx.x; item < nv * (HD / 4); item += 64 * KW) {
    const int c = item / (HD / 4), x = item % (HD / 4);
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < KW; w++) mx = fmaxf(mx, s_ml[w][c][0]);
    float den = 0.f;
    f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < KW; w++) {
      const float mw = s_ml[w][c][0], f = mw == mx ? 1.f : __builtin_amdgcn_exp2f(mw - mx);      // (all -inf: sums of zero)
      const f32x4 v = *reinterpret_cast<const f32x4*>(so + (w * nv + c) * HD + 4 * x);
      den = fmaf(f, s_ml[w][c][1], den);
#pragma unroll
      for (int i = 0; i < 4; i++) acc[i] = fmaf(f, v[i], acc[i]);
    }
    const int col = c0 + c, i = en.count == 1 ? 0 : col / a.group, h = kvh * a.group + col - i * a.group;
    if (a.splits > 1) {
      const long long rec = ((en.tok0 + i) * a.heads + h) * a.splits + split;
      *reinterpret_cast<f32x4*>(a.part + rec * HD + 4 * x) = acc;
      if (x == 0) { a.ml[rec * 2] = mx; a.ml[rec * 2 + 1] = den; }
    } else {
      const float inv = den == 0.f ? 0.f : 1.f / den;      // a row that sees nothing gives zeros
#pragma unroll
      for (int e = 0; e < 4; e++) acc[e] *= inv;
      kv4_store4<DT>(a.out, (en.tok0 + i) * a.o_ts + h * a.o_hs + 4 * x, acc, a.act16);
    }
  }
}

// a single token's key and value join the cache, by the workgroup whose pages hold its place; every thread of it comes here
template <int HD>
__device__ __forceinline__ void kv4_append_first(const Kv4Args& a, const Kv4Entry& en, const Kv4Range& rg, int kvh) {
  if (a.k != nullptr && en.count == 1 && en.start >= 0) {
    const int b = en.start >> KV4_PAGE_SHIFT;
    if (b >= rg.lo && b < rg.hi) {
      unsigned int* page = kv4_page(a, en.seq, b, kvh, HD);
      if (page && threadIdx.x < 64) kv4_append_one<HD, true>(a, page, blockIdx.z, en.tok0, en.start, kvh);
      __syncthreads();
    }
  }
}

// Few columns (a few tokens' query heads): the KW waves of a workgroup divide the keys, wave w the blocks w, w + KW, ... of the split's; all columns in each.
// 16 rows of up to 2000 tokens, five tokens each, 16 / 8 heads of 128: 13 us (1.9 TB/s), a way of eight blocks a wave between its start and the meeting of the waves.
template <int HD, int NT, int KW, int QT, int TQ, int TP>
__global__ __launch_bounds__(64 * KW) void kv4_attend_keys_kernel(const Kv4Args a) {
  typedef Kv4Sums<HD, NT, QT, TQ, TP> Sums;
  constexpr int CT = Sums::CT;
  extern __shared__ __attribute__((aligned(16))) float kv4_lds[];
  __shared__ __attribute__((aligned(16))) float s_par[KW][2 * HD];
  __shared__ float s_ml[KW][16][2];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q4 = lane >> 4, r16 = lane & 15;
  const int kvh = blockIdx.x % a.kv_heads, split = blockIdx.x / a.kv_heads;
  const Kv4Entry en = kv4_entry(a, blockIdx.z);
  const int ncol = en.count * a.group, col0 = (int)blockIdx.y * 16 * NT;
  if (col0 >= ncol) return;
  const int first = en.start + col0 / a.group, last = en.start + min(col0 + 16 * NT - 1, ncol - 1) / a.group;      // positions of the columns
  const Kv4Range rg = kv4_range(first, last, a.window, a.table_len, split, a.splits);
  if (NT == 1) kv4_append_first<HD>(a, en, rg, kvh);
  const int key_lo = a.window > 0 ? max(0, first - a.window + 1) : 0;
  const int b_hi = min(rg.hi * 4, (last >> 5) + 1), b_lo = max(rg.lo * 4, key_lo >> 5);
  Sums s;
  s.start(a, en, kvh, col0, ncol, q4, r16);
  s.template all<KW>(a, en.seq, kvh, b_lo + wv, b_hi, first, last, s_par[wv], lane);
  s.finish(q4);
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const int c0 = col0 + 16 * t, nv = min(16, ncol - c0);
    if (nv <= 0) break;
    if (t > 0) __syncthreads();
    if (q4 == 0) { s_ml[wv][r16][0] = s.m[t] * a.scale_log2; s_ml[wv][r16][1] = s.l[t]; }
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int c = 4 * q4 + r;
      if (c < nv)
#pragma unroll
        for (int x = 0; x < CT; x++) kv4_lds[(wv * nv + c) * HD + 16 * x + r16] = s.o[t][x][r];
    }
    __syncthreads();
    kv4_meet<HD, KW, QT>(a, en, kvh, split, c0, nv, kv4_lds, s_ml);
  }
}

// Many columns (portions): the four waves of a workgroup divide them, 16 NT each, and walk the same keys, whose operands they make together.  Bound by the vector units, some 370 instructions a
// block of 32 tokens and 32 columns beside 52 of the matrix units: 2048 tokens behind 6144, 32 / 8 heads of 128, 487 us with their append and read-back (495 TFLOP/s).  Operands made by each wave for itself: 30 us more;
// tiles in their order, so that a compute unit gets two with many keys: 80 us more.
template <int HD, int NT, int QT, int TQ, int TP>
__global__ __launch_bounds__(256) void kv4_attend_columns_kernel(const Kv4Args a) {
  typedef Kv4Sums<HD, NT, QT, TQ, TP> Sums;
  constexpr int CT = Sums::CT;
  __shared__ __attribute__((aligned(16))) float s_par[4][2 * HD];
  __shared__ bf16x8_t s_op[2 * 2 * CT * 64];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q4 = lane >> 4, r16 = lane & 15;
  const int kvh = blockIdx.x % a.kv_heads, split = blockIdx.x / a.kv_heads;
  const Kv4Entry en = kv4_entry(a, blockIdx.z);
  // the tiles with most keys first, downwards, then those with fewest, upwards: two workgroups of a compute unit have about the same to do in sum
  const int tiles = gridDim.y, upper = (tiles + 1) / 2, tile = (int)blockIdx.y < upper ? tiles - 1 - (int)blockIdx.y : (int)blockIdx.y - upper;
  const int ncol = en.count * a.group, wg0 = tile * 64 * NT, col0 = wg0 + wv * 16 * NT;
  if (wg0 >= ncol) return;       // (the whole workgroup)
  const int first = en.start + wg0 / a.group, last = en.start + min(wg0 + 64 * NT - 1, ncol - 1) / a.group;
  const Kv4Range rg = kv4_range(first, last, a.window, a.table_len, split, a.splits);
  const int key_lo = a.window > 0 ? max(0, first - a.window + 1) : 0;
  const int b_hi = min(rg.hi * 4, (last >> 5) + 1), b_lo = max(rg.lo * 4, key_lo >> 5);
  Sums s;
  s.start(a, en, kvh, col0, ncol, q4, r16);
  const int until = en.start + min(col0 + 16 * NT - 1, ncol - 1) / a.group;
  int w0, w1;
  Sums::whole(a, b_hi, first, last, w0, w1);
  s.template walk_shared<false>(a, en.seq, kvh, max(b_lo, w0), w1, 0, 0, col0 < ncol, until, s_op, s_par[wv], wv, lane);
  s.template walk_shared<true>(a, en.seq, kvh, b_lo, b_hi, w0, w1, col0 < ncol, until, s_op, s_par[wv], wv, lane);
  s.finish(q4);
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const int mine = col0 + 16 * t + r16;
    if (a.splits > 1 && mine < ncol && q4 == 0) {
      const long long rec = ((en.tok0 + mine / a.group) * a.heads + kvh * a.group + mine % a.group) * a.splits + split;
      a.ml[rec * 2] = s.m[t] * a.scale_log2;
      a.ml[rec * 2 + 1] = s.l[t];
    }
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int c = col0 + 16 * t + 4 * q4 + r;
      const float den = __shfl(s.l[t], 4 * q4 + r, 64);
      if (c >= ncol) continue;
      const int i = c / a.group, h = kvh * a.group + c - i * a.group;
      if (a.splits > 1) {
        float* dst = a.part + (((en.tok0 + i) * a.heads + h) * a.splits + split) * HD;
#pragma unroll
        for (int x = 0; x < CT; x++) dst[16 * x + r16] = s.o[t][x][r];
      } else {
        const float inv = den == 0.f ? 0.f : 1.f / den;
        const long long at = (en.tok0 + i) * a.o_ts + h * a.o_hs;
#pragma unroll
        for (int x = 0; x < CT; x++) kv4_store1<QT>(a.out, at + 16 * x + r16, s.o[t][x][r] * inv, a.act16);
      }
    }
  }
}

// Single tokens of up to RPT query heads a key / value head (4 or 8).  S = Q K^T the other way round: rows query heads, columns tokens, and the 16 rows are the heads 16 / RPT times
// over, so that the products of 16 / RPT tiles of tokens give every lane the scores of one token for four heads (quarter q takes its rows from the product of tile q, or q / 2): a lane
// reads the parameters of its own token, and each score, exponential and weight is worked out once and not for 16 columns of which RPT are asked for.  The weights
// pass through LDS into the A operand of P V (rows heads).  What a row's four heads share (references, their sums' factors) is the same in every lane that holds the row.
// Memory and vector units overlap but for a fifth: 32 rows of up to 4096 tokens, 32 / 8 heads of 128, 25.2 us (4.0 TB/s; 19 to 21 without the arithmetic), one of 131071 with 64 / 8 heads 34.0
// (4.4 TB/s; 25).  Short rows are one dependent way, table, page, sums: 713 tokens, 7.1 us (3.7 without the arithmetic).
template <int HD, int RPT, int KW, int QT, int TQ, int TP>
__global__ __launch_bounds__(64 * KW) void kv4_attend_token_kernel(const Kv4Args a) {
  constexpr int G = HD / 64, CH = HD / 32, CT = HD / 16, PARTS = HD / 64, PW = HD / 32;
  constexpr int NJ = 16 / RPT, TOK = 16 * NJ, NB = TOK / 32;      // tiles, tokens and blocks of a step
  constexpr int WS = TOK + 8;                                     // a head's weights in LDS, padded by 16 bytes
  extern __shared__ __attribute__((aligned(16))) float kv4_lds[];
  __shared__ __attribute__((aligned(16))) unsigned short s_w[KW][TP][RPT][WS];      // one group's weights, in the order of the value words' tokens
  __shared__ float s_ml[KW][16][2];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q4 = lane >> 4, n16 = lane & 15;
  const int kvh = blockIdx.x % a.kv_heads, split = blockIdx.x / a.kv_heads;
  const Kv4Entry en = kv4_entry(a, blockIdx.z);
  if (en.count < 1) return;
  const int last = en.start;
  const Kv4Range rg = kv4_range(last, last, a.window, a.table_len, split, a.splits);
  kv4_append_first<HD>(a, en, rg, kvh);
  const int key_lo = a.window > 0 ? max(0, last - a.window + 1) : 0;
  const int b_hi = min(rg.hi * 4, (last >> 5) + 1), b_lo = max(rg.lo * 4, key_lo >> 5) & ~(NB - 1);      // (a step's blocks are of one page)
  const int tile = RPT == 4 ? q4 : q4 >> 1;                       // this lane's token of a step: 16 tile + n16, heads h0 .. h0 + 3
  const int h0 = RPT == 4 ? 0 : 4 * (q4 & 1);
  u32x4 rk[NB][PARTS] = {}, rv[NB][PARTS] = {};                   // a step's codes (of no block: numbers too) and its token's parameters
  unsigned int rp[PW] = {};
  const unsigned int* heads = a.pool + (size_t)kvh * (36 * HD);
  const size_t page_words = (size_t)a.kv_heads * (36 * HD);
  auto load_keys = [&](int id, int b) {
    const unsigned int* blk = heads + id * page_words + (size_t)(b & 3) * kv4_block_words<HD>();
#pragma unroll
    for (int x = 0; x < NB; x++)
#pragma unroll
      for (int i = 0; i < PARTS; i++) rk[x][i] = load_nt(reinterpret_cast<const u32x4*>(blk + x * kv4_block_words<HD>()) + i * 64 + lane);
    const unsigned int* pw = blk + (tile >> 1) * kv4_block_words<HD>() + 8 * HD + (16 * (tile & 1) + n16) * PW;
    if constexpr (PW == 4) { const u32x4 w = load_nt(reinterpret_cast<const u32x4*>(pw)); rp[0] = w[0]; rp[1] = w[1]; rp[2] = w[2]; rp[3] = w[3]; }
    else { const u32x2 w = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(pw)); rp[0] = w[0]; rp[1] = w[1]; }
  };
  auto load_values = [&](int id, int b) {
    const unsigned int* blk = heads + id * page_words + (size_t)(b & 3) * kv4_block_words<HD>() + 4 * HD;
#pragma unroll
    for (int x = 0; x < NB; x++)
#pragma unroll
      for (int i = 0; i < PARTS; i++) rv[x][i] = load_nt(reinterpret_cast<const u32x4*>(blk + x * kv4_block_words<HD>()) + i * 64 + lane);
  };
  constexpr int STEP = KW * NB;
  int b = b_lo + wv * NB, id0 = kv4_page_id(a, en.seq, b, b_hi), id1 = kv4_page_id(a, en.seq, b + STEP, b_hi);
  if (id0 >= 0) { load_keys(id0, b); load_values(id0, b); }
  // queries: row n16 = head n16 % RPT, channels 32 c + 8 q .. + 7; the sums of a group's channels per head of this lane
  bf16x8_t qf[CH][TQ];
  float qs[G][4];
  {
    const long long base = en.tok0 * a.q_ts + (kvh * a.group + min(n16 % RPT, a.group - 1)) * a.q_hs + 8 * q4;
    float sum[G];
#pragma unroll
    for (int g = 0; g < G; g++) sum[g] = 0.f;
#pragma unroll
    for (int ch = 0; ch < CH; ch++) {
      float x[8];
      kv4_load8<QT>(a.q, base + 32 * ch, x);
#pragma unroll
      for (int e = 0; e < 8; e++) x[e] *= a.q_sign;
#pragma unroll
      for (int term = 0; term < TQ; term++) {
        u32x4 f;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          f[e] = pack_bf16(x[kv4_slot[2 * e]], x[kv4_slot[2 * e + 1]]);
          sum[ch / 2] += bf16_lo(f[e]) + bf16_hi(f[e]);
          x[kv4_slot[2 * e]] -= bf16_lo(f[e]); x[kv4_slot[2 * e + 1]] -= bf16_hi(f[e]);
        }
        qf[ch][term] = __builtin_bit_cast(bf16x8_t, f);
      }
    }
#pragma unroll
    for (int g = 0; g < G; g++) {
      const float t = kv4_sum_quarters(sum[g]);
#pragma unroll
      for (int r = 0; r < 4; r++) qs[g][r] = __shfl(t, h0 + r, 64);
    }
  }
  f32x4 o[CT];
  float m[4], ref[4], l[4], lov[G][4];                            // references of the weights, in scores before the scale and (ref) negative behind it
#pragma unroll
  for (int r = 0; r < 4; r++) {
    m[r] = -INFINITY; ref[r] = INFINITY; l[r] = 0.f;
#pragma unroll
    for (int g = 0; g < G; g++) lov[g][r] = 0.f;
  }
#pragma unroll
  for (int c = 0; c < CT; c++) o[c] = f32x4{0.f, 0.f, 0.f, 0.f};
  // a head's sum over the lanes that hold its tokens
  auto over_tokens = [&](float v) {
    v = row_group_sum<16>(v);
    u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
    v = __uint_as_float(w[0]) + __uint_as_float(w[1]);
    if constexpr (RPT == 4) { w = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false)); v = __uint_as_float(w[0]) + __uint_as_float(w[1]); }
    return v;
  };
  // the part of the los joins o: rows 0 .. RPT - 1 of the sums are in quarter(s) 0 (and 1), as this lane's heads there
  auto fold = [&] {
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
      for (int g = 0; g < G; g++) {
        const float t = over_tokens(lov[g][r]);
        lov[g][r] = 0.f;
#pragma unroll
        for (int c = 0; c < 4; c++) o[4 * g + c][r] += t;
      }
  };
  const int w_at = (tile >> 1) * 32 + (n16 >> 2) * 8 + 2 * (n16 & 3) + (tile & 1);      // this lane's token among a head's weights
  const float scale = a.scale_log2, gap = a.gap;
  int steps = 0;

  // Steps: NB blocks each; what is not seen (or there) has levels of zero and a score of -inf.  The next step's keys are asked for when this one's are products, its values behind
  // P V, the page of the step behind in front of both: one set of registers, and no branch around the sums.
  for (; b < b_hi; b += STEP) {
    const int id2 = kv4_page_id(a, en.seq, b + 2 * STEP, b_hi);
    const int j = b * KV4_BLK + 16 * tile + n16;
    const bool in = id0 >= 0 && j >= key_lo && j <= last;
    float st[2][G], lo[2][G];
#pragma unroll
    for (int w = 0; w < PW; w++) {
      const unsigned int x = in ? rp[w] : 0u;
      st[w / G][w % G] = bf16_hi(x); lo[w / G][w % G] = bf16_lo(x);
    }
    const float begin = in ? 0.f : -INFINITY;
    float sc[4];
#pragma unroll
    for (int g = 0; g < G; g++) {
      f32x4 d[NJ];
#pragma unroll
      for (int t = 0; t < NJ; t++) {
        d[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 2; c++) {
          const int x = (t & 1) * CH + 2 * g + c;
          const bf16x8_t kf = kv4_frag(rk[t >> 1][x >> 2][x & 3]);
#pragma unroll
          for (int term = 0; term < TQ; term++) d[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(qf[2 * g + c][term], kf, d[t], 0, 0, 0);
        }
      }
#pragma unroll
      for (int r = 0; r < 4; r++) {
        float v;
        if constexpr (RPT == 4) v = q4 < 2 ? (q4 == 0 ? d[0][r] : d[1][r]) : (q4 == 2 ? d[NJ - 2][r] : d[NJ - 1][r]);
        else v = q4 < 2 ? d[0][r] : d[1][r];
        sc[r] = fmaf(st[0][g], v, fmaf(lo[0][g], qs[g][r], g == 0 ? begin : sc[r]));
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (id1 >= 0) load_keys(id1, b + STEP);
    if (__any(sc[0] > m[0] + gap || sc[1] > m[1] + gap || sc[2] > m[2] + gap || sc[3] > m[3] + gap)) {
#pragma unroll
      for (int r = 0; r < 4; r++) {
        float mx = fmaxf(sc[r], m[r]);
        mx = fmaxf(mx, dpp_mov<0xB1, 0xf>(mx));
        mx = fmaxf(mx, dpp_mov<0x4E, 0xf>(mx));
        mx = fmaxf(mx, dpp_mov<0x141, 0xf>(mx));
        mx = fmaxf(mx, dpp_mov<0x140, 0xf>(mx));
        u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false));
        mx = fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1]));
        if constexpr (RPT == 4) {
          w = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(__float_as_uint(mx), __float_as_uint(mx), false, false));
          mx = fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1]));
        }
        const float f = mx > m[r] ? kv4_factor(m[r], mx, scale) : 1.f;
        m[r] = mx; ref[r] = -mx * scale;
        l[r] *= f;
#pragma unroll
        for (int g = 0; g < G; g++) lov[g][r] *= f;
#pragma unroll
        for (int c = 0; c < CT; c++) o[c][r] *= f;
      }
    }
    float p[4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
      p[r] = __builtin_amdgcn_exp2f(fmaf(sc[r], scale, ref[r]));
      if (!in) p[r] = 0.f;                                        // (a reference of -inf: nothing was seen yet)
      l[r] += p[r];
    }
#pragma unroll
    for (int g = 0; g < G; g++) {
      float ps[4];
#pragma unroll
      for (int r = 0; r < 4; r++) { ps[r] = p[r] * st[1][g]; lov[g][r] = fmaf(p[r], kv4_base<TP>(lo[1][g], st[1][g]), lov[g][r]); }
#pragma unroll
      for (int term = 0; term < TP; term++) {
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          const unsigned int w = pack_bf16(ps[r], ps[r + 1]);
          s_w[wv][term][h0 + r][w_at] = (unsigned short)w;
          s_w[wv][term][h0 + r + 1][w_at] = (unsigned short)(w >> 16);
          if (term + 1 < TP) { ps[r] -= bf16_lo(w); ps[r + 1] -= bf16_hi(w); }
        }
      }
      wave_fence();
      bf16x8_t wf[NB][TP];
#pragma unroll
      for (int x = 0; x < NB; x++)
#pragma unroll
        for (int term = 0; term < TP; term++) wf[x][term] = *reinterpret_cast<const bf16x8_t*>(&s_w[wv][term][n16 % RPT][32 * x + 8 * q4]);
      wave_fence();
      f32x4 sum[4];
#pragma unroll
      for (int c = 0; c < 4; c++) sum[c] = kv4_about_middle<TP>() ? f32x4{0.f, 0.f, 0.f, 0.f} : o[4 * g + c];
#pragma unroll
      for (int x = 0; x < NB; x++) {
        bf16x8_t vf[4];
#pragma unroll
        for (int c = 0; c < 4; c++) {
          const int i = 4 * g + c;
          vf[c] = kv4_operand<TP>(rv[x][i >> 2][i & 3]);
          sum[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[x][TP - 1], vf[c], sum[c], 0, 0, 0);
        }
#pragma unroll
        for (int term = TP - 2; term >= 0; term--)
#pragma unroll
          for (int c = 0; c < 4; c++) sum[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[x][term], vf[c], sum[c], 0, 0, 0);
      }
#pragma unroll
      for (int c = 0; c < 4; c++) {
        if constexpr (kv4_about_middle<TP>()) o[4 * g + c] += sum[c];
        else o[4 * g + c] = sum[c];
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (id1 >= 0) load_values(id1, b + STEP);
    id0 = id1; id1 = id2;
    if (!kv4_about_middle<TP>() && ++steps % (KV4_FOLD / NB) == 0) fold();
  }
  fold();
#pragma unroll
  for (int r = 0; r < 4; r++) l[r] = over_tokens(l[r]);
  const int nv = a.group;
  if (q4 < RPT / 4) {
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int c = 4 * q4 + r;
      if (c < nv) {
        if (n16 == 0) { s_ml[wv][c][0] = -ref[r]; s_ml[wv][c][1] = l[r]; }
#pragma unroll
        for (int x = 0; x < CT; x++) kv4_lds[(wv * nv + c) * HD + 16 * x + n16] = o[x][r];
      }
    }
  }
  __syncthreads();
  kv4_meet<HD, KW, QT>(a, en, kvh, split, 0, nv, kv4_lds, s_ml);
}

// The splits' records of a row (token, query head): a workgroup a row.  A chain of round trips and no more than that: sums are asked for before the weights are known, and every wave works
// out all weights (lane s the splits s, s + 64, ..), which go to their sums by lane exchange.
// 4.0 us behind an attention launch; with weights first, by way of LDS, 4.7.
template <int HD, int DT>
__global__ __launch_bounds__(256) void kv4_combine_kernel(const Kv4Args a) {
  constexpr int LN = HD / 4, WAYS = 256 / LN, PER = 64 / WAYS;      // lanes of a row, splits at a time, rounds of 64 splits
  __shared__ f32x4 sacc[256];
  const Kv4Entry en = kv4_entry(a, blockIdx.z);
  if ((int)blockIdx.y >= en.count) return;
  const int h = blockIdx.x, S = a.splits, tid = threadIdx.x, lane = tid & 63, ln = tid % LN, way = tid / LN;
  const long long row = (en.tok0 + blockIdx.y) * a.heads + h;
  const float* ml = a.ml + row * S * 2;
  const f32x4* part = reinterpret_cast<const f32x4*>(a.part + row * S * HD) + ln;
  f32x4 v[PER];
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int s = way + i * WAYS;
    v[i] = s < S ? part[(size_t)s * LN] : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  float w[4], l[4], mx = -INFINITY, tot = 0.f;                       // (at most 256 splits)
#pragma unroll
  for (int q = 0; q < 4; q++) {
    const int s = lane + 64 * q;
    w[q] = s < S ? ml[2 * s] : -INFINITY;
    l[q] = s < S ? ml[2 * s + 1] : 0.f;
    mx = fmaxf(mx, w[q]);
  }
  mx = fmaxf(mx, dpp_mov<0xB1, 0xf>(mx));
  mx = fmaxf(mx, dpp_mov<0x4E, 0xf>(mx));
  mx = fmaxf(mx, dpp_mov<0x141, 0xf>(mx));
  mx = fmaxf(mx, dpp_mov<0x140, 0xf>(mx));
  mx = kv4_max_quarters(mx);
#pragma unroll
  for (int q = 0; q < 4; q++) {
    w[q] = w[q] == mx ? 1.f : __builtin_amdgcn_exp2f(w[q] - mx);
    tot = fmaf(w[q], l[q], tot);
  }
  tot = kv4_sum_quarters(row_group_sum<16>(tot));
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int q = 0; q < 4; q++) {
    if (64 * q >= S) break;
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const int s = 64 * q + way + i * WAYS;
      if (q > 0) v[i] = s < S ? part[(size_t)s * LN] : f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const float f = __shfl(w[q], way + i * WAYS, 64);
#pragma unroll
      for (int c = 0; c < 4; c++) acc[c] = fmaf(f, v[i][c], acc[c]);
    }
  }
  sacc[tid] = acc;
  __syncthreads();
  if (tid < LN) {
#pragma unroll
    for (int k = 1; k < WAYS; k++) {
      const f32x4 o = sacc[k * LN + tid];
#pragma unroll
      for (int c = 0; c < 4; c++) acc[c] += o[c];
    }
    const float inv = tot == 0.f ? 0.f : 1.f / tot;
    const long long at = (en.tok0 + blockIdx.y) * a.o_ts + h * a.o_hs + 4 * tid;
#pragma unroll
    for (int c = 0; c < 4; c++) acc[c] *= inv;
    kv4_store4<DT>(a.out, at, acc, a.act16);
  }
}

// ---- page copies --------------------------------------------------------------------------------------------------------------------------------------
struct CopyPagesArgs {
  const unsigned char* src; unsigned char* dst;
  long long src_pool, dst_pool, page;                         // bytes between the pools of two layers, and of a page (a multiple of 16)
  long long src_pages, dst_pages;                             // pages of a pool
  const int *from, *to; int n;                                // pairs; one outside of its pool is left out
};
// a workgroup a (16 KB piece of a page, pair, layer): memory's rate, 180 pages of 147 KB in 32 layers 317 us (5.4 TB/s, reads and writes; a copy of 1 GiB has 5.0); a page in 16 layers 3.4 us
constexpr int COPY_PIECE = 16384;
static __global__ __launch_bounds__(256) void copy_pages_kernel(const CopyPagesArgs a) {
  const int pair = blockIdx.y;
  const long long f = a.from[pair], t = a.to[pair];
  if (f < 0 || f >= a.src_pages || t < 0 || t >= a.dst_pages) return;
  const long long p0 = (long long)blockIdx.x * COPY_PIECE;
  const u32x4* s = reinterpret_cast<const u32x4*>(a.src + blockIdx.z * a.src_pool + f * a.page + p0);
  u32x4* d = reinterpret_cast<u32x4*>(a.dst + blockIdx.z * a.dst_pool + t * a.page + p0);
  const long long left = (a.page - p0) / 16;
  const int n = (int)(left < COPY_PIECE / 16 ? left : COPY_PIECE / 16);
  u32x4 v[4];
#pragma unroll
  for (int i = 0; i < 4; i++) { const int x = threadIdx.x + 256 * i; if (x < n) v[i] = load_nt(s + x); }
#pragma unroll
  for (int i = 0; i < 4; i++) { const int x = threadIdx.x + 256 * i; if (x < n) __builtin_nontemporal_store(v[i], d + x); }
}

}  // namespace tgx
