// The 4-bit KV cache format: quantising a row, storing it, reading it back.
//
// A value is scale * code + minimum, code in 0..15, with one bf16 (minimum, scale) pair per group of
// 32, 64 or 128 consecutive dimensions of one token's K (or V) row.  For a group with minimum m and
// maximum M (exact, the inputs are bf16):
//   scale = bf16((M - m) * fp32(1/15)), 0 if that is below 2^-126
//   code  = floor(min((v - m) * (1 / scale) + (1/2 + 2^-12), 15.5)), every step in fp32; 0 if scale = 0
// The 2^-12 sends ties (v half way between two codes, frequent since v and scale have 8 significant
// bits each) up whatever the rounding of the reciprocal.  A row that holds a NaN or an infinity, or a
// group whose M - m overflows, is stored with scale = minimum = NaN in all its groups: it reads back as
// NaN instead of as finite values it never held.
//
// A page is page_size / 16 records of 16 tokens.  A record is
//   [K codes 8 D][K pairs 64 NG][V codes 8 D][V pairs 64 NG] bytes, NG = D / group,
// pairs token-major, minimum in the low half of the 32-bit pair.  The codes are laid out so that the lanes
// of a warp get whole mma.m16n8k16 A fragments by 16-byte (D = 128) or 8-byte (D = 64) accesses with no
// shuffle and no shared-memory bank conflict (lane = 4 g + t4, word j holds dimensions 32 j ..):
//   K: token r, byte r D/2 + t4 D/8 + 4 j: the 8 codes of dimensions 32 j + 8 t4 ..
//   V: byte half 4 D + (4 g + t4) D/8 + 4 j: the 4 codes of dimensions 32 j + 4 g .. of token
//      8 half + 2 t4 (low 16 bits) and of token 8 half + 2 t4 + 1 (high 16 bits)
// No two tokens share a byte, so rows are written independently of one another.
#pragma once

#include "common.cuh"

namespace wgkv {

template <int D, int NG>
struct Kv4 {
  static constexpr int kWords = D / 32;              // 32-bit words of codes per lane and row
  static constexpr int kRow = D + 8 * NG;            // bytes of a token (K and V)
  static constexpr int kRec = 16 * kRow;             // bytes of a record
  static constexpr int kKP = 8 * D;                  // offsets in a record: K pairs, V codes, V pairs
  static constexpr int kV = 8 * D + 64 * NG;
  static constexpr int kVP = 16 * D + 64 * NG;
};

// Tensor-side description of a cache and of the heads' pages (device pointers).
struct Kv4Pages {
  uint8_t* data;
  int64_t num_pages;
  int page;            // tokens per page, a multiple of 16
  const int32_t* table;
  int64_t table_stride;
  int width;           // pages a table row lists
  int* err;
};

// The record of token position `pos` of head row `bh` (0 <= pos < width * page), or NULL with an error
// flagged when the table names no page of the cache there.
template <int D, int NG>
WGKV_DEV uint8_t* kv4_record(const Kv4Pages& c, int64_t bh, int pos) {
  const int pid = __ldg(c.table + bh * c.table_stride + pos / c.page);
  if (pid < 0 || pid >= c.num_pages) {
    set_error(c.err, WGKV_ERR_BAD_PAGE);
    return nullptr;
  }
  return c.data + (int64_t(pid) * (c.page >> 4) + (pos % c.page >> 4)) * Kv4<D, NG>::kRec;
}

WGKV_DEV uint32_t bf2_min(uint32_t a, uint32_t b) {  // NaN-propagating, per half
  const __nv_bfloat162 r = __hmin2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
WGKV_DEV uint32_t bf2_max(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Quantises the rows a warp holds, four lanes to a row: lane t of a row has raw[j] = its bf16 values of
// dimensions 32 j + 8 t .. + 7.  Gives the lane's words of codes (word j: those 8, low code first) and
// the row's pairs (in all four lanes).  All lanes of the warp call it.
template <int D, int NG>
WGKV_DEV void kv4_quantise(const uint4* raw, uint32_t* words, uint32_t* pairs) {
  constexpr int W = D / 32, PG = W / NG;  // words per group
  const int lane = threadIdx.x & 31;
  float lo[NG], inv[NG], sc[NG];
  bool bad = false;
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    uint32_t a = raw[n * PG].x, z = a;
#pragma unroll
    for (int j = n * PG; j < (n + 1) * PG; ++j) {
      a = bf2_min(bf2_min(a, raw[j].x), bf2_min(bf2_min(raw[j].y, raw[j].z), raw[j].w));
      z = bf2_max(bf2_max(z, raw[j].x), bf2_max(bf2_max(raw[j].y, raw[j].z), raw[j].w));
    }
    // (min, -) and (max, -) of the two halves, then over the row's four lanes
    a = bf2_min(a, a >> 16 | a << 16);
    z = bf2_max(z, z >> 16 | z << 16);
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      const uint32_t m = (a & 0xffffu) | (z << 16);
      const uint32_t p = __shfl_xor_sync(0xffffffff, m, o);
      a = bf2_min(a, p & 0xffffu | p << 16);
      z = bf2_max(z, p >> 16 | p & 0xffff0000u);
    }
    lo[n] = __uint_as_float(a << 16);
    const float range = __uint_as_float(z << 16) - lo[n];
    bad |= !(range <= 3.402823466e38f);
    float s = bf16_round(__fmul_rn(range, 1.f / 15.f));
    if (!(s >= 1.17549435e-38f)) s = 0.f;
    sc[n] = s;
    inv[n] = s > 0.f ? __frcp_rn(s) : 0.f;
  }
  // one bad group spoils the whole row
  const uint32_t votes = __ballot_sync(0xffffffff, bad);
  bad = (votes >> (lane & 28)) & 15u;
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    pairs[n] = bad ? 0x7fc07fc0u : __float_as_uint(sc[n]) | (__float_as_uint(lo[n]) >> 16);
#pragma unroll
    for (int j = n * PG; j < (n + 1) * PG; ++j) {
      const uint32_t u[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
      uint32_t w = 0;
#pragma unroll
      for (int e = 7; e >= 0; --e) {
        const float v = e & 1 ? __uint_as_float(u[e >> 1] & 0xffff0000u) : __uint_as_float(u[e >> 1] << 16);
        // (M - m) / scale is at most 15 (1 + 2^-8), so the bound 15.5 holds by itself.  Fusing the product
        // and the sum changes no code: where v - m is a multiple of the scale's last bit, the quotient is
        // 2^-17 or more (relative) away from where the code steps, 32 times fp32's roundings.
        const float t = __fmaf_rn(__fsub_rn(v, lo[n]), inv[n], 0.5f + 0.000244140625f);
        // adding 2^23 rounding down leaves floor(t) in the low bits: 0x4b000000 + code
        w = w * 16u + __float_as_uint(__fadd_rd(t, 8388608.f));
      }
      w -= 0xfb000000u;  // 0x4b000000 * 0x11111111 mod 2^32
      words[j] = bad ? 0u : w;
    }
  }
}

template <int W>
WGKV_DEV void st_words(uint8_t* p, const uint32_t* w) {
  if (W == 4) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
}

template <int NG>
WGKV_DEV void kv4_store_pairs(uint8_t* p, int t, const uint32_t* pairs) {
  if (t >= NG) return;
  uint32_t x = pairs[0];
#pragma unroll
  for (int n = 1; n < NG; ++n) x = t == n ? pairs[n] : x;
  reinterpret_cast<uint32_t*>(p)[t] = x;
}

// Lane t (0..3) of a row stores its K words and the row's pairs at place r (0..15) of a record.
template <int D, int NG>
WGKV_DEV void kv4_store_k(uint8_t* rec, int r, int t, const uint32_t* words, const uint32_t* pairs) {
  st_words<D / 32>(rec + r * (D / 2) + t * (D / 8), words);
  kv4_store_pairs<NG>(rec + Kv4<D, NG>::kKP + r * 4 * NG, t, pairs);
}

// The same for a V row.  `both`: lane ^ 4 of the warp stores place r ^ 1 of the same record, so the two
// lanes swap halves and store whole words; otherwise the row goes out in 2-byte pieces.  All lanes of
// the warp call it; `valid` lanes store, and `both` is the same in the two lanes.
template <int D, int NG>
WGKV_DEV void kv4_store_v(uint8_t* rec, int r, int t, const uint32_t* words, const uint32_t* pairs, bool valid,
                          bool both) {
  constexpr int W = D / 32;
  uint32_t lo[W / 2], hi[W / 2];  // 16-bit halves of two words: dimension chunks g = 2 t and 2 t + 1
#pragma unroll
  for (int i = 0; i < W / 2; ++i) {
    lo[i] = __byte_perm(words[2 * i], words[2 * i + 1], 0x5410);
    hi[i] = __byte_perm(words[2 * i], words[2 * i + 1], 0x7632);
  }
  const int odd = r & 1;
  uint8_t* base = rec + Kv4<D, NG>::kV + (r >> 3) * 4 * D + ((r & 7) >> 1) * (D / 8);
  uint32_t out[W];
#pragma unroll
  for (int i = 0; i < W / 2; ++i) {  // the even place takes chunk 2 t, the odd one chunk 2 t + 1
    const uint32_t got = __shfl_xor_sync(0xffffffff, odd ? lo[i] : hi[i], 4);
    const uint32_t a = odd ? got : lo[i], b = odd ? hi[i] : got;
    out[2 * i] = __byte_perm(a, b, 0x5410);
    out[2 * i + 1] = __byte_perm(a, b, 0x7632);
  }
  if (!valid) return;
  if (both) {
    st_words<W>(base + (2 * t + odd) * 4 * (D / 8), out);
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) {
      uint8_t* p = base + 2 * t * 4 * (D / 8) + 4 * j + 2 * odd;
      *reinterpret_cast<uint16_t*>(p) = uint16_t(words[j]);
      *reinterpret_cast<uint16_t*>(p + 4 * (D / 8)) = uint16_t(words[j] >> 16);
    }
  }
  kv4_store_pairs<NG>(rec + Kv4<D, NG>::kVP + r * 4 * NG, t, pairs);
}

template <int W>
WGKV_DEV void ld_words(uint32_t* w, const uint8_t* p) {
  if (W == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  }
}

// The words and pairs of lane t of the K (or V) row at place r of a record: kv4_store_k / _v undone.
template <int D, int NG>
WGKV_DEV void kv4_load_k(const uint8_t* rec, int r, int t, uint32_t* words, uint32_t* pairs) {
  ld_words<D / 32>(words, rec + r * (D / 2) + t * (D / 8));
#pragma unroll
  for (int n = 0; n < NG; ++n) pairs[n] = reinterpret_cast<const uint32_t*>(rec + Kv4<D, NG>::kKP + r * 4 * NG)[n];
}

template <int D, int NG>
WGKV_DEV void kv4_load_v(const uint8_t* rec, int r, int t, uint32_t* words, uint32_t* pairs) {
  constexpr int W = D / 32;
  const uint8_t* base = rec + Kv4<D, NG>::kV + (r >> 3) * 4 * D + ((r & 7) >> 1) * (D / 8) + 2 * t * 4 * (D / 8);
  uint32_t a[W], b[W];
  ld_words<W>(a, base);
  ld_words<W>(b, base + 4 * (D / 8));
#pragma unroll
  for (int j = 0; j < W; ++j) words[j] = __byte_perm(a[j], b[j], r & 1 ? 0x7632 : 0x5410);
#pragma unroll
  for (int n = 0; n < NG; ++n) pairs[n] = reinterpret_cast<const uint32_t*>(rec + Kv4<D, NG>::kVP + r * 4 * NG)[n];
}

// Value of a code: the product is exact (8 + 4 significant bits), the sum rounds once.
WGKV_DEV float kv4_value(uint32_t code, uint32_t pair) {
  return fmaf(__uint_as_float(pair & 0xffff0000u), float(code), __uint_as_float(pair << 16));
}

// One warp quantises the row of a new token (k and v: D bf16 each, 4-byte aligned) into place r of a
// record: lanes 0-3 take K, lanes 4-7 V.
template <int D, int NG>
WGKV_DEV void kv4_put_row(uint8_t* rec, int r, const uint16_t* k, const uint16_t* v) {
  constexpr int W = D / 32;
  const int lane = threadIdx.x & 31, t = lane & 3;
  uint4 raw[W];
#pragma unroll
  for (int j = 0; j < W; ++j) {
    raw[j] = make_uint4(0, 0, 0, 0);
    if (lane < 8) {
      const uint32_t* src = reinterpret_cast<const uint32_t*>((lane < 4 ? k : v) + 32 * j + 8 * t);
      raw[j] = make_uint4(src[0], src[1], src[2], src[3]);
    }
  }
  uint32_t words[W], pairs[NG];
  kv4_quantise<D, NG>(raw, words, pairs);
  if (lane < 4) kv4_store_k<D, NG>(rec, r, t, words, pairs);
  kv4_store_v<D, NG>(rec, r, t, words, pairs, lane >= 4 && lane < 8, false);
}

// Calls f.run<D, NG>() for a supported (head_dim, group); false otherwise.
template <typename F>
__host__ __device__ inline bool kv4_dispatch(int head_dim, int group, F&& f) {
  if (head_dim == 128) {
    if (group == 32) return f.template run<128, 4>(), true;
    if (group == 64) return f.template run<128, 2>(), true;
    if (group == 128) return f.template run<128, 1>(), true;
  } else if (head_dim == 64) {
    if (group == 32) return f.template run<64, 2>(), true;
    if (group == 64) return f.template run<64, 1>(), true;
  }
  return false;
}

inline bool kv4_supported(int head_dim, int group) {
  return (head_dim == 64 || head_dim == 128) && (group == 32 || group == 64 || group == 128) && group <= head_dim;
}

}  // namespace wgkv
