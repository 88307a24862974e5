// Writing rows into the 4-bit KV cache and reading them back (format: kv4.cuh).
//
// Both are one pass over the data and bound by HBM: a token costs 4 D bytes of bf16 and D + 8 D / group of
// codes.  Measured on B200, D = 128, groups of 64, 64K rows of 8 heads (343 MB each way), in replayed graphs:
// writing 62 us, 5.5 TB/s, 0.84 of the copy bandwidth (66 us by itself on cold data, with 0.77 of the issue slots
// busy: 102 warp instructions a row, 5 per value and lane: unpack, subtract, multiply-add, round down, shift in);
// reading 53 us, 6.5 TB/s, 0.99 (54 us by itself).
#include <type_traits>
#include <utility>

#include "kv4.cuh"
#include "runtime.h"

namespace wgkv {
namespace {

struct Kv4Rows {  // (B, Hk, L, D) bf16 with element strides
  const uint16_t* p;
  int64_t sb, sh, st;
};

// Rows r of head bh go to positions start[bh] + r, r < min(counts[bh], L).  A warp takes 8 positions
// aligned to 8 (so that the two tokens which share 32-bit words of V codes meet in one warp), four lanes
// to a row, each with 16-byte pieces of it: a row's loads and its K and V codes are whole sectors.
template <int D, int NG, bool kVec16>
__global__ void __launch_bounds__(256) kv4_append_kernel(Kv4Pages c, Kv4Rows K, Kv4Rows V, int Hk, int L,
                                                         const int32_t* start, const int32_t* counts) {
  constexpr int W = D / 32;
  const int bh = blockIdx.y, b = bh / Hk, h = bh - b * Hk;
  const int lane = threadIdx.x & 31, t = lane & 3;
  const int64_t first = __ldg(start + bh);
  const int64_t n = counts ? min(max(__ldg(counts + bh), 0), L) : L;
  const int64_t pos = (first & ~int64_t(7)) + (int64_t(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5)) * 8 +
                      (lane >> 2);
  const int64_t r = pos - first;
  bool valid = r >= 0 && r < n;
  if (!__any_sync(0xffffffff, valid)) return;
  const int place = int(pos) & 15;
  uint4 kr[W], vr[W];
#pragma unroll
  for (int j = 0; j < W; ++j) {
    kr[j] = vr[j] = make_uint4(0, 0, 0, 0);
    if (valid) {
      const uint16_t* ks = K.p + b * K.sb + h * K.sh + r * K.st + 32 * j + 8 * t;
      const uint16_t* vs = V.p + b * V.sb + h * V.sh + r * V.st + 32 * j + 8 * t;
      if (kVec16) {
        kr[j] = __ldg(reinterpret_cast<const uint4*>(ks));
        vr[j] = __ldg(reinterpret_cast<const uint4*>(vs));
      } else {
        uint32_t kw[4], vw[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          kw[e] = __ldg(ks + 2 * e) | uint32_t(__ldg(ks + 2 * e + 1)) << 16;
          vw[e] = __ldg(vs + 2 * e) | uint32_t(__ldg(vs + 2 * e + 1)) << 16;
        }
        kr[j] = make_uint4(kw[0], kw[1], kw[2], kw[3]);
        vr[j] = make_uint4(vw[0], vw[1], vw[2], vw[3]);
      }
    }
  }
  uint8_t* rec = nullptr;  // looked up while the rows arrive
  if (valid) {
    if (pos < 0 || pos >= int64_t(c.width) * c.page) set_error(c.err, WGKV_ERR_HEAD_CAPACITY);
    else rec = kv4_record<D, NG>(c, bh, int(pos));
    valid = rec != nullptr;
  }
  uint32_t words[W], pairs[NG];
  kv4_quantise<D, NG>(kr, words, pairs);
  if (valid) kv4_store_k<D, NG>(rec, place, t, words, pairs);
  kv4_quantise<D, NG>(vr, words, pairs);
  const bool both = __shfl_xor_sync(0xffffffff, int(valid), 4) && valid;
  kv4_store_v<D, NG>(rec, place, t, words, pairs, valid, both);
}

// out[bh, i] = the row at position start[bh] + i for i < min(counts[bh], rows), zeros behind it: four
// lanes to a row, every store instruction of a warp writes eight 64-byte pieces.
template <int D, int NG>
__global__ void __launch_bounds__(256) kv4_read_kernel(Kv4Pages c, const int32_t* start, const int32_t* counts,
                                                       int rows, uint16_t* out_k, uint16_t* out_v) {
  constexpr int W = D / 32;
  const int bh = blockIdx.y, lane = threadIdx.x & 31, t = lane & 3;
  const int64_t i = (int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5)) * 8 + (lane >> 2);
  if (i >= rows) return;
  const int n = min(__ldg(counts + bh), rows);
  const uint8_t* rec = nullptr;
  int64_t pos = 0;
  if (i < n) {
    pos = (start ? __ldg(start + bh) : 0) + i;
    if (pos < 0 || pos >= int64_t(c.width) * c.page) set_error(c.err, WGKV_ERR_HEAD_CAPACITY);
    else rec = kv4_record<D, NG>(c, bh, int(pos));
  }
  uint32_t kw[W], vw[W], kp[NG], vp[NG];
#pragma unroll
  for (int j = 0; j < W; ++j) kw[j] = vw[j] = 0;
#pragma unroll
  for (int g = 0; g < NG; ++g) kp[g] = vp[g] = 0;
  if (rec) {
    kv4_load_k<D, NG>(rec, int(pos) & 15, t, kw, kp);
    kv4_load_v<D, NG>(rec, int(pos) & 15, t, vw, vp);
  }
  const int64_t at = (int64_t(bh) * rows + i) * D + 8 * t;
#pragma unroll
  for (int j = 0; j < W; ++j) {
    uint32_t ko[4], vo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t kpair = kp[j * NG / W], vpair = vp[j * NG / W];
      ko[e] = pack_bf16x2(kv4_value((kw[j] >> (8 * e)) & 15u, kpair), kv4_value((kw[j] >> (8 * e + 4)) & 15u, kpair));
      vo[e] = pack_bf16x2(kv4_value((vw[j] >> (8 * e)) & 15u, vpair), kv4_value((vw[j] >> (8 * e + 4)) & 15u, vpair));
    }
    *reinterpret_cast<uint4*>(out_k + at + 32 * j) = make_uint4(ko[0], ko[1], ko[2], ko[3]);
    *reinterpret_cast<uint4*>(out_v + at + 32 * j) = make_uint4(vo[0], vo[1], vo[2], vo[3]);
  }
}

struct AppendLaunch {
  Kv4Pages c;
  Kv4Rows K, V;
  int Hk, BH, L;
  const int32_t *start, *counts;
  bool vec16;
  cudaStream_t stream;
  template <int D, int NG>
  void run() {
    const int warps = (L + 7 + 7) / 8;  // 8-aligned windows that L rows can touch
    const int per = warps < 8 ? warps : 8;
    const dim3 grid((warps + per - 1) / per, BH);
    if (vec16) kv4_append_kernel<D, NG, true><<<grid, 32 * per, 0, stream>>>(c, K, V, Hk, L, start, counts);
    else kv4_append_kernel<D, NG, false><<<grid, 32 * per, 0, stream>>>(c, K, V, Hk, L, start, counts);
  }
};

struct ReadLaunch {
  Kv4Pages c;
  int BH, rows;
  const int32_t *start, *counts;
  uint16_t *out_k, *out_v;
  cudaStream_t stream;
  template <int D, int NG>
  void run() {
    kv4_read_kernel<D, NG><<<dim3((rows + 63) / 64, BH), 256, 0, stream>>>(c, start, counts, rows, out_k, out_v);
  }
};

bool pages_ok(const void* cache, int64_t num_pages, int page_size, const int32_t* table, int64_t table_stride,
              int table_width) {
  return cache && (reinterpret_cast<uintptr_t>(cache) & 15) == 0 && num_pages > 0 && page_size > 0 &&
         page_size % 16 == 0 && table && table_width > 0 && table_stride >= table_width &&
         int64_t(table_width) * page_size < (int64_t(1) << 31);
}

}  // namespace
}  // namespace wgkv

using namespace wgkv;

extern "C" int wgkv_kv4_row_bytes(int head_dim, int group) {
  return kv4_supported(head_dim, group) ? head_dim + 8 * (head_dim / group) : WGKV_EINVAL;
}

extern "C" int wgkv_kv4_append(const uint16_t* k, int64_t k_sb, int64_t k_sh, int64_t k_st, const uint16_t* v,
                               int64_t v_sb, int64_t v_sh, int64_t v_st, int batch, int kv_heads, int rows,
                               int head_dim, int group, uint8_t* cache, int64_t num_pages, int page_size,
                               const int32_t* start, const int32_t* counts, const int32_t* block_table,
                               int64_t table_stride, int table_width, int* err, void* stream) {
  if (!kv4_supported(head_dim, group) ||
      !pages_ok(cache, num_pages, page_size, block_table, table_stride, table_width))
    return WGKV_EINVAL;
  if (!k || !v || !start || batch <= 0 || kv_heads <= 0 || rows < 0 || int64_t(batch) * kv_heads > 65535)
    return WGKV_EINVAL;
  if (rows == 0) return WGKV_OK;
  const bool vec16 = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0 &&
                     (k_sb | k_sh | k_st | v_sb | v_sh | v_st) % 8 == 0;
  AppendLaunch a{{cache, num_pages, page_size, block_table, table_stride, table_width, err},
                 {k, k_sb, k_sh, k_st}, {v, v_sb, v_sh, v_st}, kv_heads, batch * kv_heads, rows, start, counts, vec16,
                 as_stream(stream)};
  kv4_dispatch(head_dim, group, a);
  return cudaGetLastError() == cudaSuccess ? WGKV_OK : WGKV_ECUDA;
}

extern "C" int wgkv_kv4_read(const uint8_t* cache, int64_t num_pages, int page_size, int head_dim, int group,
                             const int32_t* start, const int32_t* counts, const int32_t* block_table,
                             int64_t table_stride, int table_width, int batch, int kv_heads, int rows,
                             uint16_t* out_k, uint16_t* out_v, int* err, void* stream) {
  if (!kv4_supported(head_dim, group) ||
      !pages_ok(cache, num_pages, page_size, block_table, table_stride, table_width))
    return WGKV_EINVAL;
  if (!counts || !out_k || !out_v || batch <= 0 || kv_heads <= 0 || rows < 0 || int64_t(batch) * kv_heads > 65535 ||
      ((reinterpret_cast<uintptr_t>(out_k) | reinterpret_cast<uintptr_t>(out_v)) & 15))
    return WGKV_EINVAL;
  if (rows == 0) return WGKV_OK;
  ReadLaunch a{{const_cast<uint8_t*>(cache), num_pages, page_size, block_table, table_stride, table_width, err},
               batch * kv_heads, rows, start, counts, out_k, out_v, as_stream(stream)};
  kv4_dispatch(head_dim, group, a);
  return cudaGetLastError() == cudaSuccess ? WGKV_OK : WGKV_ECUDA;
}

namespace {

// Slot i of an argument array as a T.
template <typename T>
T slot(const void* slots, int i) {
  const int64_t v = static_cast<const int64_t*>(slots)[i];
  if constexpr (std::is_pointer<T>::value) return reinterpret_cast<T>(static_cast<intptr_t>(v));
  else return static_cast<T>(v);
}

// the one floating argument travels as a double
template <>
float slot<float>(const void* slots, int i) {
  return static_cast<float>(static_cast<const double*>(slots)[i]);
}

template <typename... Args, int... I>
int call(int (*fn)(Args...), const void* slots, std::integer_sequence<int, I...>) {
  return fn(slot<Args>(slots, I)...);
}

template <typename... Args>
int call(int (*fn)(Args...), const void* slots) {
  return call(fn, slots, std::make_integer_sequence<int, int(sizeof...(Args))>());
}

}  // namespace

extern "C" int wgkv_kv4_call(int op, const void* slots) {
  if (!slots) return WGKV_EINVAL;
  switch (op) {
    case WGKV_KV4_APPEND: return call(wgkv_kv4_append, slots);
    case WGKV_KV4_READ: return call(wgkv_kv4_read, slots);
    case WGKV_KV4_PAGED_DECODE: return call(wgkv_paged_decode_kv4, slots);
    default: return WGKV_EINVAL;
  }
}

extern "C" uint64_t wgkv_stream_capture_id(void* stream) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (cudaStreamGetCaptureInfo(as_stream(stream), &status, &id) != cudaSuccess) {
    cudaGetLastError();  // the legacy stream beside another stream's capture: not captured itself
    return 0;
  }
  return status == cudaStreamCaptureStatusActive ? id : 0;
}
