// Ragged paged decode attention over a 4-bit KV cache (format: kv4.cuh), sm_100a.
//
// With K = s_k c + m_k and V = s_v c + m_v per group of dimensions (c the codes, s and m the group's scale
// and minimum), for every token t and query head h
//   x_th = scale (sum_g s_k[t,g] (q_hg . c_tg) + m_k[t,g] (1 . q_hg)),
//   out_h = (sum_t p_th s_v[t,g] c_t + sum_t p_th m_v[t,g]) / sum_t p_th,   p = 2^(x - reference),
// so the matrix products run on the codes themselves and no value is ever expanded:
//
// * Tokens are the M side of both products (mma.m16n8k16, fp16 in, fp32 accumulate): S^T = C_k Q^T and
//   O^T = C_v^T P^T with 8 query heads as N.  Up to 8 query heads per KV head take 16 instructions per 16
//   tokens at D = 128, half of what heads on the M side (16 rows, mostly padding) would.
// * A code is an fp16 operand without conversion: masked out of its word it is the subnormal code * 2^-24
//   (bits 0-3) or code * 2^-20 (bits 4-7), which the tensor cores multiply exactly.  The factors are
//   undone on q (odd k-steps carry q / 16) and on the output (odd m-tiles).  5 integer operations unpack
//   8 codes of K.  V takes 4: its even m-tiles get both codes of a byte, low + 16 high, and the odd ones'
//   sums are subtracted at the end (in fp32, 17 times the low codes' rounding).
// * q enters as fp16 times a power of two per head that puts its largest element in [2^14, 2^15): exact
//   down to 2^-24 of it, 2^-36 of it absolute below.
// * The weights p s_v are rounded to fp16: to 11 bits from 2^-14 up, to multiples of 2^-24 below.  The
//   reference 2^r of p is a running maximum over x + exponent(s_v), not over x, so that the weights, not the
//   probabilities, have the same largest size however V's scale differs between tokens.  It is the token's
//   largest scale that counts, so the weights of a group with smaller scales, and those of a long tail behind
//   one heavy token, lie below: the largest weight is settled at 2^7 and the reference moves only when one
//   would pass 2^15.5, near the end of fp16's range, which leaves 20 bits below the largest weight for the
//   smaller ones to be normal numbers in, and 31 until they vanish (settled at 1, 7 fewer, groups 2^-12 apart
//   behind a token 8 nats above the rest were lost).  Exponents below -40 count as -40.  Sums of p
//   and p m_v stay fp32.
// * The tensor cores' fp32 accumulation truncates.  Sums of codes, all positive, lose up to 2^-23 of
//   themselves with every record added, and V's that cancel (any long, flat softmax) leave a result
//   hundreds of times smaller than the sums: 8e-3 of it was lost at 28K tokens.  So every record's (or
//   pair of records') products start from zero and join O^T by paired fp32 additions, which round to
//   nearest.
// * With up to 4 query heads per KV head, two records share the 8 columns (kPack = 2): columns 0-3 hold the
//   heads' scores for the tokens of the first, columns 4-7 for those of the second, so that the softmax, the
//   scales and the weights of both are one set of instructions instead of two half-empty ones; the weights
//   are masked per record before the second product, and the two softmax states become one where the head
//   ends (105 us -> 97 us at 3.5M tokens x heads).
// * S^T's accumulators hold a token per lane row, P^T's fragment a head per lane row: movmatrix turns the
//   packed weights, one per 8x8 block.
//
// Work is cut as in paged_decode.cu: the 16-token records of all heads laid end to end, equal segments per
// CTA; a head cut over CTAs is merged by the last one to finish it (self-resetting counter, fixed order of
// summation).  Heads stand apart in that line by what the end of one costs (kHeadCost): the CTAs with most
// heads' ends in their segments had finished up to 20 % later than the others.  Inside a CTA every warp is on
// its own: it takes every kWarps-th pair of records of the segment's part of a head, copies them itself
// (cp.async.bulk, one whole record each) into a ring of slots of its own, a pair each, and works on a pair at a
// time; page ids are looked up 32 records at a time, a batch ahead.  Warps meet only where a head ends.
// Measured and not taken: one producer warp for all and a stage shared by all warps (112 us against 102 then);
// one warp merging the states while the others go on with the next head (100 against 97); the join of partial
// results fed by bulk copies into shared memory (25 against 21 us with 8 heads of 16 rows).  The copies alone,
// without any arithmetic, take 85 us.
//
// Measured on B200: 3.5M tokens x KV heads (G = 4, D = 128, groups of 64, 504 MB) in 98 us by itself with nothing
// of them in L2, 5.1 TB/s, 0.79 of the copy bandwidth, and 91 us a call in a replayed graph of 20 calls, whose set-up
// overlaps the call before and finds a part of the data in L2; the bf16 kernel takes 287 us on the same tokens (1.79
// GB).  The times by which variants are compared in this file are of such graphs.  What bounds it there is latency
// with 3 warps per scheduler (168 registers): 223 instructions a record, 72 of them unpacking, at 0.51 of the issue
// slots and 0.57 of the integer pipe.  A single sequence of 2K tokens takes 9.0 us, all of it latency: four dependent
// look-ups (lengths, table, records; then the counter and the partial results) of 0.4 to 1 us each around one pair
// of records per warp.
//
// The launch is a programmatic dependent one whatever pdl_enabled() says of the others: set-up overlaps the kernel
// before, and the queries, lengths and tables are read behind griddep_wait().  It never cost (a step of a 4-bit
// Llama-3.1-8B shape in graph replay 3.99 ms with, 4.00 without; Llama-3.2-1B 1.090 with, 1.100 without; append and
// attention of 32 sequences 60.6 with, 61.3 us without).

#include <algorithm>

#include "kv4.cuh"
#include "runtime.h"

namespace wgkv {
namespace {

constexpr int kNB = 2;         // records of a slot, which a warp works on together
constexpr int kSlots = 2;      // slots of a warp's ring (3: 1-2 % slower at every size)
constexpr int kLaneHeads = 8;  // heads per lane up to which a warp sums up all lengths itself
constexpr int kMaxBH = 4096;
constexpr int kMaxG = 16;

// 12 warps of 168 registers on an SM: 6 in each of two CTAs, and 4 in each of three where there are many heads,
// whose ends a CTA of fewer warps gets over sooner (256 heads and more: 16 -> 15 us and 56 -> 54 us, 512: 17.4
// -> 16.1 us and 70 -> 67 us; 32 heads: 11.5 -> 12.5 us, 40 -> 40.5 us), and all in one where there are few heads
// of more than 4 rows, whose partial results are then half as many (2 heads, 16K tokens: 15.1 -> 12.3 us, 16 heads,
// 30K: 21.0 -> 18.8 us; 64 heads, 4K: 14.3 -> 14.5 us; with up to 4 rows 8 heads of 2K: 8.7 -> 9.7 us).  16 warps of
// 128 registers spill (100 us against 90.5 at 3.5M tokens x heads).
constexpr int kSmWarps = 12, kManyHeads = 256, kFewHeads = 64;
// A CTA that meets a head's end before its segment's spends about as long on the merge and the next head's
// start as on kHeadCost records: the heads stand that far apart in the line.  Segments are cut at the heads'
// ends where that makes them no more than kAlignSlack records longer.
constexpr int kHeadCost = 40;
constexpr int kAlignSlack = 16;
// Exponents (of two) of the weights: where the largest is settled, and which one moves the reference.  A weight is
// below 2^1.5 times what its exponent says (scales up to 2, the exponent's sum rounded to an integer), and fp16
// ends at 2^16.
constexpr float kSettled = 7.f, kLargest = 14.f;

struct Kv4DecodeParams {
  Kv4Pages c;
  const uint16_t* q;
  uint16_t* out;
  const int32_t* seqlens;
  int group;      // query heads per KV head
  int halves;     // 1 where a KV head's query heads are worked on as two heads of up to 8 (else 0)
  int BH, G;      // heads worked on, query heads of each (one fewer in a second half, if group is odd)
  int slots;      // kSlots: as a constant it costs registers (91 -> 93 us at 3.5M tokens x heads)
  float scale_log2;
  float* part;    // partial results: (BH + CTAs) x G x (D + 4)
  int* counters;  // per head
};

WGKV_DEV void mma_f16_16816(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same onto zero.
WGKV_DEV void mma_f16_16816_first(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                  uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// Two fp32 values in a register pair, added and multiplied by one instruction each (same roundings).
WGKV_DEV uint64_t f2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
WGKV_DEV float f2_get(uint64_t v, int i) { return __uint_as_float(uint32_t(v >> (32 * i))); }
WGKV_DEV uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
WGKV_DEV uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

WGKV_DEV uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

WGKV_DEV uint32_t movmatrix_trans(uint32_t a) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}

WGKV_DEV float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <bool kB>
struct Whole {
  static constexpr bool value = kB;
};

// N words from shared memory at byte address a (a multiple of 4 N).  The "memory" clobbers of the barrier
// waits around them keep these loads in their stage.
template <int N>
WGKV_DEV void lds_words(uint32_t* w, uint32_t a) {
  if (N == 4)
    asm("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1 % N]), "=r"(w[2 % N]), "=r"(w[3 % N]) : "r"(a) : "memory");
  else if (N == 2)
    asm("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1 % N]) : "r"(a) : "memory");
  else
    asm("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(a) : "memory");
}

// One look at a barrier's phase; most pairs have arrived when they are asked for.
WGKV_DEV bool mbar_done(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n"
      " mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done;
}

// The rest of a wait, with its limit; once one of a CTA has run into it the others do not wait at all.
__device__ __noinline__ void wait_longer(uint64_t* bar, uint32_t parity, volatile int* gave_up, int* err) {
  if (*gave_up || mbar_wait(bar, parity)) return;
  *gave_up = 1;
  set_error(err, WGKV_ERR_TIMEOUT);
}

template <int D>
__host__ __device__ constexpr int merge_row() { return D + 4; }  // D values, maximum, sum; rows 16 bytes apart mod 128

// What sums relative to reference m are worth relative to M >= m.
WGKV_DEV float factor(float m, float M) { return m == M ? 1.f : exp2_approx(m - M); }

// Counts one more, ordered behind this thread's view of memory and ahead of what it reads next (two fences
// around a relaxed atomic take 0.4 us longer).
WGKV_DEV int count_up(int* p) {
  int old;
  asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(old) : "l"(p) : "memory");
  return old;
}

// (A, L) += f (a, l).
WGKV_DEV void add_state(float4& A, float& L, float f, const float4& a, float l) {
  L = fmaf(f, l, L);
  A.x = fmaf(f, a.x, A.x), A.y = fmaf(f, a.y, A.y), A.z = fmaf(f, a.z, A.z), A.w = fmaf(f, a.w, A.w);
}

// Four output values A / L; a head whose scores are all NaN has L = NaN.
WGKV_DEV void store_out(uint16_t* out, const float4& A, float L) {
  *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16x2(A.x / L, A.y / L), pack_bf16x2(A.z / L, A.w / L));
}

size_t fixed_smem(int warps, int BH, int G, int D) {
  return 128 + size_t(warps) * (G * (D + 4) * 4 + 32 * 32 + kSlots * 8) +
         size_t(2 * BH + (32 + 2) * warps) * 4 + 64;
}

// Tokens of head bh that count: not below 0, not past the table.
WGKV_DEV int head_len(const Kv4DecodeParams& p, int bh) {
  return min(max(__ldg(p.seqlens + (bh >> p.halves)), 0), p.c.width * p.c.page);
}

// ceil(n / d) for 0 <= n < 2^29 + 2^20, d > 0 and a quotient below 2^22 (the line's records over 148 CTAs at
// least, or a number of CTAs): __fdividef is off by up to 2 ulps, 1/2 at such quotients, and n by up to 32 in fp32,
// less than 1/4 over the CTAs, so the fp32 quotient is at most one off.
WGKV_DEV int ceil_div(int n, int d) {
  n += d - 1;
  int q = int(__fdividef(float(n), float(d)));
  const int r = n - q * d;
  return r < 0 ? q - 1 : r >= d ? q + 1 : q;
}

// The first query head (row of q and out) of head bh.
WGKV_DEV size_t query_row(const Kv4DecodeParams& p, int bh) {
  return size_t(bh >> p.halves) * p.group + (bh & p.halves) * p.G;
}

// kPack: records whose scores share the 8 columns of a tile: 2 for up to 4 query heads, else 1.
template <int D, int NG, int kPack, int kWarps>
__global__ void __launch_bounds__(32 * kWarps, kSmWarps / kWarps) kv4_decode_kernel(Kv4DecodeParams p) {
  constexpr int kThreads = 32 * kWarps;
  constexpr int kMinSegment = kWarps * kNB;  // records a CTA gets at least
  using F = Kv4<D, NG>;
  constexpr int kSets = kNB / kPack;  // sets of columns that a pair of records fills
  constexpr int W = D / 32;
  constexpr int kMR = merge_row<D>();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* stage_base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
  const int R = p.slots;
  const int G = p.G, BH = p.BH;
  float* merge = reinterpret_cast<float*>(stage_base + size_t(kWarps) * R * kNB * F::kRec);  // [kWarps][G][kMR]
  float* join = merge + kWarps * G * kMR;                                                  // [kThreads][8]
  uint64_t* bars = reinterpret_cast<uint64_t*>(join + kThreads * 8);                        // [kWarps][kSlots]
  int* pre = reinterpret_cast<int*>(bars + kWarps * kSlots);  // [BH] a head's first record in the line
  int* fin = pre + BH;                                           // [BH] the one behind its last
  int* scan = fin + BH;                                          // [kThreads]
  int* flag = scan + kThreads + 2 * kWarps;
  volatile int* gave_up = flag + 1;  // a wait of this CTA ran into its limit

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffff, tid >> 5, 0);  // the same in all lanes, so branches on it are uniform
  const uint32_t ring = smem_u32(stage_base) + warp * R * kNB * F::kRec;
  uint64_t* full = bars + warp * kSlots;
  if (lane < R) mbar_init(&full[lane], kNB);
  fence_barrier_init();
  *gave_up = 0;
  griddep_wait();  // lengths, tables and rows may come from the launch just before
  griddep_launch();

  // ---- the line of all heads' records and its cut into segments of `seg`, one per CTA ----
  int seg, u0, u1, lo;
  if (BH <= 32 * kLaneHeads) {
    // each warp for itself (all write the same values): no barrier between the launch and the first copy
    const int per = (BH + 31) >> 5;
    int n[kLaneHeads], room[kLaneHeads], sum = 0;
    bool over = false;
#pragma unroll
    for (int k = 0; k < kLaneHeads; ++k) {
      const int i = lane * per + k;
      const int len = k < per && i < BH ? __ldg(p.seqlens + (i >> p.halves)) : 0;
      over |= len > p.c.width * p.c.page;
      n[k] = (min(max(len, 0), p.c.width * p.c.page) + 15) >> 4;
    }
    if (over && blockIdx.x == 0) set_error(p.c.err, WGKV_ERR_HEAD_CAPACITY);
#pragma unroll
    for (int k = 0; k < kLaneHeads; ++k) sum += n[k];
    const int U = __reduce_add_sync(0xffffffff, sum);
    int longest = 0;
#pragma unroll
    for (int k = 0; k < kLaneHeads; ++k) longest = max(longest, n[k]);
    longest = __reduce_max_sync(0xffffffff, longest);
    // A partial result of G x D values costs the CTA that joins them about as long as G x D / 900 records: as
    // many records to a segment, at least, as the partial results of the longest head are worth (2 KV heads of
    // 8 query heads, 16K tokens: 20.8 -> 15.1 us).
    const int worth = int(sqrtf(float(longest) * float(G * D) * (1.f / 900.f)));
    const int least = max(max(kMinSegment, worth), ceil_div(U, gridDim.x));
    // segments that end with the heads, if slightly longer ones are then few enough
    seg = 0;
    if (ceil_div(U, least + kAlignSlack) + BH / 2 <= int(gridDim.x)) {
      for (int more = 0; more <= kAlignSlack; more += more ? more : 2) {
        const int longer = least + more;
        int cut[kLaneHeads], ctas = 0;
#pragma unroll
        for (int k = 0; k < kLaneHeads; ++k) {
          cut[k] = 0;
          if (k < per) cut[k] = ceil_div(n[k], longer);
          ctas += cut[k];
        }
        if (__reduce_add_sync(0xffffffff, ctas) > int(gridDim.x)) continue;
        seg = longer;
        sum = 0;
#pragma unroll
        for (int k = 0; k < kLaneHeads; ++k) {
          room[k] = cut[k] * seg;
          sum += room[k];
        }
        break;
      }
    }
    if (seg == 0) {
      sum = 0;
#pragma unroll
      for (int k = 0; k < kLaneHeads; ++k) {
        room[k] = n[k] ? n[k] + kHeadCost : 0;
        sum += room[k];
      }
      seg = max(least, ceil_div(__reduce_add_sync(0xffffffff, sum), gridDim.x));
    }
    int run = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffff, run, o);
      if (lane >= o) run += y;
    }
    const int line = __shfl_sync(0xffffffff, run, 31);
    run -= sum;
    u0 = min(line, int(blockIdx.x) * seg);
    u1 = min(line, u0 + seg);
    int before = 0;  // heads that begin at or before u0
#pragma unroll
    for (int k = 0; k < kLaneHeads; ++k) {
      const int i = lane * per + k;
      if (k < per && i < BH) {
        pre[i] = run;
        fin[i] = run + n[k];
        before += run <= u0;
      }
      run += room[k];
    }
    lo = __reduce_add_sync(0xffffffff, before) - 1;
    __syncwarp();
  } else {
    const int per = (BH + kThreads - 1) / kThreads;
    const int i0 = min(BH, tid * per), i1 = min(BH, i0 + per);
    int sum = 0, U;
    for (int i = i0; i < i1; ++i) {
      const int n = (head_len(p, i) + 15) >> 4;
      sum += n ? n + kHeadCost : 0;
      if (blockIdx.x == 0 && __ldg(p.seqlens + (i >> p.halves)) > p.c.width * p.c.page)
        set_error(p.c.err, WGKV_ERR_HEAD_CAPACITY);
    }
    int run = block_excl_scan<kThreads>(sum, scan, U);
    for (int i = i0; i < i1; ++i) {
      const int n = (head_len(p, i) + 15) >> 4;
      pre[i] = run;
      fin[i] = run + n;
      run += n ? n + kHeadCost : 0;
    }
    seg = max(kMinSegment, ceil_div(U, gridDim.x));
    u0 = min(U, int(blockIdx.x) * seg);
    u1 = min(U, u0 + seg);
    __syncthreads();
    int hi = BH;  // pre[lo] <= u0, and u0 < pre[hi] if there is a head hi
    lo = 0;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= u0) lo = mid;
      else hi = mid;
    }
  }
  auto rows_of = [&](int bh) { return min(G, p.group - (bh & p.halves) * G); };  // query heads of head bh
  for (int bh = blockIdx.x; bh < BH; bh += gridDim.x) {  // heads that hold nothing
    if (fin[bh] == pre[bh])
      for (int e = tid; e < rows_of(bh) * D; e += kThreads) p.out[query_row(p, bh) * D + e] = 0;
  }
  if (u0 >= u1) return;

  // the queries of the first head are on their way while its pages are looked up
  const int g = lane >> 2, t4 = lane & 3;
  // kPack = 2: columns 0-3 are the heads for the first record of a pair, columns 4-7 for the second
  const int half = kPack == 2 ? t4 >> 1 : 0;
  const uint32_t own[2] = {g < 4 ? 0xffffffffu : 0u, g < 4 ? 0u : 0xffffffffu};
  uint4 raw_q[W];
  auto load_q = [&](int bh) {
    const int head = kPack == 2 ? g & 3 : g;
    const uint16_t* src = p.q + (query_row(p, bh) + head) * D + 8 * t4;
#pragma unroll
    for (int j = 0; j < W; ++j)
      raw_q[j] = head < rows_of(bh) ? __ldg(reinterpret_cast<const uint4*>(src + 32 * j)) : make_uint4(0, 0, 0, 0);
  };
  while (lo < BH && fin[lo] <= max(u0, pre[lo])) ++lo;  // past heads that end before, or hold nothing
  if (lo == BH || pre[lo] >= u1) return;
  load_q(lo);

  // ---- this warp's records in order: of the pairs of each head's part of the segment, every kWarps-th ----
  const int upp = p.c.page >> 4;
  int2* from = reinterpret_cast<int2*>(scan + kThreads) + warp;  // the next batch starts at this warp's pair
  if (lane == 0) *from = make_int2(lo, 0);                       // from->y of head from->x's part
  int f_page = 0, f_rec = -1;  // this lane's record of the batch fetched last: page id, as looked up, and place in it
  auto fetch = [&]() {         // 16 pairs, a record per lane (f_rec -1 for none); nothing here waits for the lookup
    __syncwarp();
    int h = from->x, o = from->y + (lane >> 1);
    f_rec = -1;
    while (h < BH && pre[h] < u1) {
      const int first = max(pre[h], u0), last = min(fin[h], u1);
      const int pairs = max(last - first + 1, 0) >> 1;  // of all warps
      const int c = (pairs - warp + kWarps - 1) / kWarps;
      if (o < c) {
        const int u = first + 2 * (warp + kWarps * o) + (lane & 1);
        if (u < last) {
          const uint32_t ul = u - pre[h], pg = upp == 1 ? ul : ul / uint32_t(upp);
          f_page = __ldg(p.c.table + int64_t(h >> p.halves) * p.c.table_stride + pg);
          f_rec = ul - pg * upp;
        }
        break;
      }
      o -= c;
      ++h;
    }
    __syncwarp();
    if (lane == 31) *from = make_int2(h, o + 1);
  };
  auto resolve = [&]() -> int {  // its place in the cache, in records
    if (f_rec < 0) return -1;
    if (f_page < 0 || f_page >= p.c.num_pages) {
      set_error(p.c.err, WGKV_ERR_BAD_PAGE);
      f_page = 0;
    }
    return f_page * upp + f_rec;
  };
  fetch();
  int batch = resolve(), used = 0;
  int slot_in = 0;
  auto issue = [&]() {  // the next pair into slot slot_in
    const int at = __shfl_sync(0xffffffff, batch, used + (lane & 1));
    if (lane < kNB && !*gave_up) {  // a slot whose copies never came is not armed again
      if (at >= 0) {
        mbar_arrive_expect_tx(&full[slot_in], F::kRec);
        bulk_load(stage_base + size_t((warp * R + slot_in) * kNB + lane) * F::kRec, p.c.data + int64_t(at) * F::kRec,
                  F::kRec, &full[slot_in]);
      } else {
        mbar_arrive(&full[slot_in]);  // a pair of one record, or none
      }
    }
    slot_in = slot_in + 1 == R ? 0 : slot_in + 1;
    used += 2;
    if (used == 32) {
      batch = resolve();
      fetch();
      used = 0;
    }
  };
  for (int i = 0; i < R; ++i) issue();
  fetch();

  int slot = 0;       // the next pair's
  uint32_t ph = 0;
  for (int bh = lo; bh < BH && pre[bh] < u1; ++bh) {
    const int hs = pre[bh], he = fin[bh];
    const int rs = max(hs, u0), re = min(he, u1);
    if (re <= rs) continue;

    // ---- queries: B fragments, power of two, sums over each group ----
    uint32_t qf[W][4];       // [word of K][even k-step b0, b1, odd k-step b0, b1]
    float qs[NG][2];         // scale_log2 * sum of the group's q, heads 2 t4 and 2 t4 + 1 of the tile
    float alpha[2];          // what a product of codes and fragments is times x's scale
    float qv[W][8];
    float big = 0.f;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      unpack8(raw_q[j], qv[j]);
#pragma unroll
      for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(qv[j][e]));
    }
    big = fmaxf(big, __shfl_xor_sync(0xffffffff, big, 1));
    big = fmaxf(big, __shfl_xor_sync(0xffffffff, big, 2));
    // 2^(14 - exponent(big)), it and its inverse times 2^24 kept normal numbers: smaller exponents count
    // as -112; a query of 2^118 or more overflows (to NaN)
    const int ex = min(max(int(__float_as_uint(big) >> 23) - 127, -112), 117);
    const float up = __uint_as_float(uint32_t(14 - ex + 127) << 23);
    float sum[NG];
#pragma unroll
    for (int n = 0; n < NG; ++n) sum[n] = 0.f;
#pragma unroll
    for (int j = 0; j < W; ++j) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sum[j * NG / W] += qv[j][e];
        qv[j][e] *= up;
      }
      qf[j][0] = pack_f16x2(qv[j][0], qv[j][4]);
      qf[j][1] = pack_f16x2(qv[j][2], qv[j][6]);
      qf[j][2] = pack_f16x2(qv[j][1] * 0.0625f, qv[j][5] * 0.0625f);
      qf[j][3] = pack_f16x2(qv[j][3] * 0.0625f, qv[j][7] * 0.0625f);
    }
    // 2^24 (the codes') / up (the queries'), as 2^(24 - 14 + ex): the lanes of heads 2 t4 and 2 t4 + 1 have it
    const float a = p.scale_log2 * __uint_as_float(uint32_t(10 + ex + 127) << 23);
#pragma unroll
    for (int c = 0; c < 2; ++c) alpha[c] = __shfl_sync(0xffffffff, a, (2 * t4 + c) * 4);
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      sum[n] += __shfl_xor_sync(0xffffffff, sum[n], 1);
      sum[n] += __shfl_xor_sync(0xffffffff, sum[n], 2);
      sum[n] *= p.scale_log2;
#pragma unroll
      for (int c = 0; c < 2; ++c) qs[n][c] = __shfl_sync(0xffffffff, sum[n], (2 * t4 + c) * 4);
    }

    uint64_t acc[2 * W][2];  // O^T: m-tile, row g and g + 8, heads 2 t4 and 2 t4 + 1 as an fp32 pair
    float um[NG][2];         // sum of p m_v over this lane's tokens
    float mx[2], l[2];
#pragma unroll
    for (int m = 0; m < 2 * W; ++m) acc[m][0] = acc[m][1] = 0;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      mx[c] = 0.f;
      l[c] = 0.f;
#pragma unroll
      for (int n = 0; n < NG; ++n) um[n][c] = 0.f;
    }

    bool first = true;  // no reference yet
    struct Scores {
      float v[kSets][4];
    };
    // 2^23 + biased exponent of the largest scale of the V rows (at least -40) of tokens g and g + 8: added to x
    // it rounds it to an integer, close enough for a bound
    auto exponents = [&](uint32_t rec) {
      uint32_t vp0[NG], vp1[NG];
      lds_words<NG>(vp0, rec + F::kVP + g * 4 * NG);
      lds_words<NG>(vp1, rec + F::kVP + (g + 8) * 4 * NG);
      uint32_t v0 = uint32_t(127 - 40) << 23, v1 = v0;
#pragma unroll
      for (int n2 = 0; n2 < NG; ++n2) {
        v0 = max(v0, vp0[n2]);
        v1 = max(v1, vp1[n2]);
      }
      return make_float2(__uint_as_float(0x4b000000u | v0 >> 23), __uint_as_float(0x4b000000u | v1 >> 23));
    };
    // Scores of a pair of records relative to the reference, and a bound of their weights.  kAll: both are
    // there and every token counts, so that nothing branches.
    auto scores = [&](uint32_t recs, auto all, int nb, int left, Scores& x, float (&top)[2]) {
      constexpr bool kAll = decltype(all)::value;
      top[0] = top[1] = -INFINITY;
#pragma unroll
      for (int i = 0; i < kSets; ++i) {
        if (!kAll && i >= nb) {
          x.v[i][0] = x.v[i][1] = x.v[i][2] = x.v[i][3] = -INFINITY;
          continue;
        }
        uint32_t k0[kPack][W], k1[kPack][W], kp0[NG], kp1[NG];
#pragma unroll
        for (int r = 0; r < kPack; ++r) {
          lds_words<W>(k0[r], recs + (i + r) * F::kRec + lane * (D / 8));
          lds_words<W>(k1[r], recs + (i + r) * F::kRec + 4 * D + lane * (D / 8));
        }
        const int mine = kPack == 2 ? half : i;  // the record whose tokens this lane's columns are about
        const uint32_t rec = recs + mine * F::kRec;
        lds_words<NG>(kp0, rec + F::kKP + g * 4 * NG);
        lds_words<NG>(kp1, rec + F::kKP + (g + 8) * 4 * NG);
        float t[4], o[4];
#pragma unroll
        for (int n2 = 0; n2 < NG; ++n2) {
          float d[kPack][4];
#pragma unroll
          for (int j = n2 * (W / NG); j < (n2 + 1) * (W / NG); ++j) {
#pragma unroll
            for (int r = 0; r < kPack; ++r) {
              const uint32_t a = k0[r][j], b = k1[r][j], a8 = a >> 8, b8 = b >> 8;
              if (j == n2 * (W / NG))
                mma_f16_16816_first(d[r], a & 0x000f000fu, b & 0x000f000fu, a8 & 0x000f000fu, b8 & 0x000f000fu,
                                    qf[j][0], qf[j][1]);
              else
                mma_f16_16816(d[r], a & 0x000f000fu, b & 0x000f000fu, a8 & 0x000f000fu, b8 & 0x000f000fu, qf[j][0],
                              qf[j][1]);
              mma_f16_16816(d[r], a & 0x00f000f0u, b & 0x00f000f0u, a8 & 0x00f000f0u, b8 & 0x00f000f0u, qf[j][2],
                            qf[j][3]);
            }
          }
          const float s0 = __uint_as_float(kp0[n2] & 0xffff0000u), m0 = __uint_as_float(kp0[n2] << 16);
          const float s1 = __uint_as_float(kp1[n2] & 0xffff0000u), m1 = __uint_as_float(kp1[n2] << 16);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float d0 = kPack == 2 && half ? d[kPack - 1][c] : d[0][c];
            const float d1 = kPack == 2 && half ? d[kPack - 1][2 + c] : d[0][2 + c];
            t[c] = n2 ? fmaf(s0, d0, t[c]) : s0 * d0;
            t[2 + c] = n2 ? fmaf(s1, d1, t[2 + c]) : s1 * d1;
            o[c] = fmaf(m0, qs[n2][c], n2 ? o[c] : -mx[c]);
            o[2 + c] = fmaf(m1, qs[n2][c], n2 ? o[2 + c] : -mx[c]);
          }
        }
        const float2 e = exponents(rec);
        const int valid = left - 16 * mine;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float y = fmaf(alpha[c & 1], t[c], o[c]);
          x.v[i][c] = kAll || g + 8 * (c >> 1) < valid ? y : -INFINITY;
        }
        top[0] = fmaxf(top[0], fmaxf(x.v[i][0] + e.x, x.v[i][2] + e.y));
        top[1] = fmaxf(top[1], fmaxf(x.v[i][1] + e.x, x.v[i][3] + e.y));
      }
    };
    // The exponent of the largest weight of each column of the warp, less where it is settled.
    auto above = [&](float (&m)[2]) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        m[c] = fmaxf(m[c], __shfl_xor_sync(0xffffffff, m[c], 4));
        m[c] = fmaxf(m[c], __shfl_xor_sync(0xffffffff, m[c], 8));
        m[c] = fmaxf(m[c], __shfl_xor_sync(0xffffffff, m[c], 16));
        m[c] -= 8388608.f + 127.f + kSettled;
      }
    };
    // Moves the reference where a weight would outgrow it: most pairs only learn that none does.
    auto settle = [&](uint32_t recs, Scores& x, const float (&top)[2]) {
      if (__any_sync(0xffffffff, first || fmaxf(top[0], top[1]) > 8388608.f + 127.f + kLargest)) {
        float by[2] = {top[0], top[1]}, fac[2];
        above(by);
        bool far = false;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          // up by `by`, where that is positive; the first time to where it belongs (a floor keeps it finite)
          by[c] = fmaxf(by[c], first ? -1e30f : 0.f);
          far |= fabsf(by[c]) > 4194304.f && fabsf(by[c]) < 1e29f;
#pragma unroll
          for (int i = 0; i < kSets; ++i) {
            x.v[i][c] -= by[c];
            x.v[i][2 + c] -= by[c];
          }
        }
        if (__any_sync(0xffffffff, far)) {
          // Scores so large that x + exponent was rounded to more than a whole number: the rest of the way from
          // what is left of them.  Without it scores of 2^29 and more can leave every weight zero or one infinite.
          float rest[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < kSets; ++i) {
            const float2 e = exponents(recs + (kPack == 2 ? half : i) * F::kRec);
#pragma unroll
            for (int c = 0; c < 2; ++c) rest[c] = fmaxf(rest[c], fmaxf(x.v[i][c] + e.x, x.v[i][2 + c] + e.y));
          }
          above(rest);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float r = by[c] != 0.f && rest[c] > -1e29f ? rest[c] : 0.f;
            by[c] += r;
#pragma unroll
            for (int i = 0; i < kSets; ++i) {
              x.v[i][c] -= r;
              x.v[i][2 + c] -= r;
            }
          }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float f = first ? 0.f : exp2_approx(-by[c]);
          mx[c] += by[c];
          l[c] *= f;
#pragma unroll
          for (int n2 = 0; n2 < NG; ++n2) um[n2][c] *= f;
          fac[c] = f;
        }
        const uint64_t both = f2(fac[0], fac[1]);
#pragma unroll
        for (int m2 = 0; m2 < 2 * W; ++m2) {
          acc[m2][0] = mul2(acc[m2][0], both);
          acc[m2][1] = mul2(acc[m2][1], both);
        }
        first = false;
      }
    };
    // Weights, and O^T += C_v^T P^T.
    auto weigh = [&](uint32_t recs, auto all, int nb, int left, const Scores& x) {
      constexpr bool kAll = decltype(all)::value;
#pragma unroll
      for (int i = 0; i < kSets; ++i) {
        if (!kAll && i >= nb) continue;
        const int mine = kPack == 2 ? half : i;
        const uint32_t rec = recs + mine * F::kRec;
        const int valid = left - 16 * mine;
        uint32_t v0[kPack][W], v1[kPack][W], vp0[NG], vp1[NG];
        lds_words<NG>(vp0, rec + F::kVP + g * 4 * NG);
        lds_words<NG>(vp1, rec + F::kVP + (g + 8) * 4 * NG);
#pragma unroll
        for (int r = 0; r < kPack; ++r) {
          lds_words<W>(v0[r], recs + (i + r) * F::kRec + F::kV + lane * (D / 8));
          lds_words<W>(v1[r], recs + (i + r) * F::kRec + F::kV + 4 * D + lane * (D / 8));
        }
        float pr[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) pr[c] = exp2_approx(x.v[i][c]);
        l[0] += pr[0] + pr[2];
        l[1] += pr[1] + pr[3];
#pragma unroll
        for (int n2 = 0; n2 < NG; ++n2) {
          if (!kAll) {  // places behind the length may hold anything
            if (g >= valid) vp0[n2] = 0;
            if (g + 8 >= valid) vp1[n2] = 0;
          }
          const float s0 = __uint_as_float(vp0[n2] & 0xffff0000u), m0 = __uint_as_float(vp0[n2] << 16);
          const float s1 = __uint_as_float(vp1[n2] & 0xffff0000u), m1 = __uint_as_float(vp1[n2] << 16);
          uint32_t pb[kPack][2];
          um[n2][0] = fmaf(pr[0], m0, fmaf(pr[2], m1, um[n2][0]));
          um[n2][1] = fmaf(pr[1], m0, fmaf(pr[3], m1, um[n2][1]));
          const uint32_t w0 = movmatrix_trans(pack_f16x2(pr[0] * s0, pr[1] * s0));
          const uint32_t w1 = movmatrix_trans(pack_f16x2(pr[2] * s1, pr[3] * s1));
#pragma unroll
          for (int r = 0; r < kPack; ++r) {  // a record's weights stand in its own columns
            pb[r][0] = kPack == 2 ? w0 & own[r] : w0;
            pb[r][1] = kPack == 2 ? w1 & own[r] : w1;
          }
#pragma unroll
          for (int j = n2 * (W / NG); j < (n2 + 1) * (W / NG); ++j) {
            float d[4], e[4];
#pragma unroll
            for (int r = 0; r < kPack; ++r) {
              // two codes at a time: even rows of O^T get low + 16 high, odd rows 16 high
              const uint32_t a = v0[r][j] & 0x00ff00ffu, b = v1[r][j] & 0x00ff00ffu;
              const uint32_t a8 = __byte_perm(v0[r][j], 0, 0x4341), b8 = __byte_perm(v1[r][j], 0, 0x4341);
              const uint32_t ah = a & 0x00f000f0u, bh16 = b & 0x00f000f0u, a8h = a8 & 0x00f000f0u, b8h = b8 & 0x00f000f0u;
              if (r == 0) {
                mma_f16_16816_first(d, a, a8, b, b8, pb[r][0], pb[r][1]);
                mma_f16_16816_first(e, ah, a8h, bh16, b8h, pb[r][0], pb[r][1]);
              } else {
                mma_f16_16816(d, a, a8, b, b8, pb[r][0], pb[r][1]);
                mma_f16_16816(e, ah, a8h, bh16, b8h, pb[r][0], pb[r][1]);
              }
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              acc[2 * j][c] = add2(acc[2 * j][c], f2(d[2 * c], d[2 * c + 1]));
              acc[2 * j + 1][c] = add2(acc[2 * j + 1][c], f2(e[2 * c], e[2 * c + 1]));
            }
          }
        }
      }
    };

    // The part's last pair (one record, perhaps, and perhaps the head's end) goes by itself.  (Taking a pair's
    // scores in one stretch of code with the weights and products of the one before: 93 us against 91.)
    const int pairs = (re - rs + 1) >> 1;
    const int mine = (pairs - warp + kWarps - 1) / kWarps;                   // this warp's
    const int whole_pairs = mine - (mine > 0 && (pairs - 1) % kWarps == warp);
    auto arrived = [&]() -> uint32_t {  // the next pair's slot, its copies landed
      if (!mbar_done(&full[slot], ph)) wait_longer(&full[slot], ph, gave_up, p.c.err);
      const uint32_t recs = ring + slot * (kNB * F::kRec);
      slot = slot + 1 == R ? 0 : slot + 1;
      ph ^= slot == 0;
      return recs;
    };
    Scores x;
    float top[2];
    for (int i = 0; i < whole_pairs; ++i) {
      const uint32_t now = arrived();
      scores(now, Whole<true>(), kNB, 0, x, top);
      settle(now, x, top);
      weigh(now, Whole<true>(), kNB, 0, x);
      __syncwarp();  // every lane has read the slot
      issue();
    }
    if (mine > whole_pairs) {
      const uint32_t now = arrived();
      const int u = rs + 2 * (pairs - 1);
      const int nb = min(kNB, re - u);
      const int left = min(head_len(p, bh) - (u - pre[bh]) * 16, 16 * nb);  // tokens of these records that count
      scores(now, Whole<false>(), nb, left, x, top);
      settle(now, x, top);
      weigh(now, Whole<false>(), nb, left, x);
      __syncwarp();
      issue();
    }

    // ---- this warp's state of the head into shared memory ----
    if constexpr (kPack == 2) {  // the two records' columns of a head (lanes t4 and t4 ^ 2) into one
      float f[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float m = fmaxf(mx[c], __shfl_xor_sync(0xffffffff, mx[c], 2));
        f[c] = factor(mx[c], m);
        mx[c] = m;
        l[c] *= f[c];
        l[c] += __shfl_xor_sync(0xffffffff, l[c], 2);
#pragma unroll
        for (int n2 = 0; n2 < NG; ++n2) {
          um[n2][c] *= f[c];
          um[n2][c] += __shfl_xor_sync(0xffffffff, um[n2][c], 2);
        }
      }
      const uint64_t both = f2(f[0], f[1]);
#pragma unroll
      for (int m = 0; m < 2 * W; ++m)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint64_t v = mul2(acc[m][c], both);
          acc[m][c] = add2(v, f2(__shfl_xor_sync(0xffffffff, f2_get(v, 0), 2),
                                    __shfl_xor_sync(0xffffffff, f2_get(v, 1), 2)));
        }
    }
    const int rows = rows_of(bh);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int head = 2 * t4 + c;
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        l[c] += __shfl_xor_sync(0xffffffff, l[c], o);
#pragma unroll
        for (int n2 = 0; n2 < NG; ++n2) um[n2][c] += __shfl_xor_sync(0xffffffff, um[n2][c], o);
      }
      if (head < rows) {
        float* row = merge + (warp * G + head) * kMR;
#pragma unroll
        for (int j = 0; j < W; ++j) {
          const float m = um[j * NG / W][c];
          const float e0 = f2_get(acc[2 * j][0], c), o0 = f2_get(acc[2 * j + 1][0], c);
          const float e1 = f2_get(acc[2 * j][1], c), o1 = f2_get(acc[2 * j + 1][1], c);
          float4 v;
          v.x = fmaf(e0 - o0, 16777216.f, m);
          v.y = fmaf(o0, 1048576.f, m);
          v.z = fmaf(e1 - o1, 16777216.f, m);
          v.w = fmaf(o1, 1048576.f, m);
          *reinterpret_cast<float4*>(row + 32 * j + 4 * g) = v;
        }
        if (g == 0) {
          row[D] = first ? -INFINITY : mx[c];
          row[D + 1] = l[c];
        }
      }
    }
    // the next head's queries on their way
    int after = bh + 1;
    while (after < BH && fin[after] == pre[after]) ++after;
    if (after < BH && pre[after] < u1) load_q(after);
    __syncthreads();

    // ---- the warps' states into one: output, or this CTA's partial result ----
    const bool whole = rs == hs && re == he;
    uint16_t* out = p.out + query_row(p, bh) * D;
    float* mine_at = p.part + size_t(bh + blockIdx.x) * G * kMR;
    for (int e = tid; e < rows * (D / 4); e += kThreads) {
      const int r = e / (D / 4), d = 4 * (e % (D / 4));
      const float* row = merge + r * kMR;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) M = fmaxf(M, row[w * G * kMR + D]);
      float L = 0.f;
      float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float* state = row + w * G * kMR;
        add_state(A, L, factor(state[D], M), *reinterpret_cast<const float4*>(state + d), state[D + 1]);
      }
      if (whole) {
        store_out(out + r * D + d, A, L);
      } else {
        *reinterpret_cast<float4*>(mine_at + r * kMR + d) = A;
        if (d == 0) *reinterpret_cast<float2*>(mine_at + r * kMR + D) = make_float2(M, L);
      }
    }
    if (!whole) {
      __syncthreads();
      const int c_first = hs / seg, np = (he - 1) / seg - c_first + 1;
      if (tid == 0) {
        const int last = count_up(&p.counters[bh]) == np - 1;  // releases what the barrier put before it
        if (last) p.counters[bh] = 0;
        *flag = last;
      }
      __syncthreads();
      if (*flag) {
        // D / 4 lanes take a query head of every `parts`-th partial result, 4 dimensions each and kChunk loads
        // in flight at once; lane i of them reads the i-th one's maximum and sum
        constexpr int kLanes = D / 4, kChunk = 16;
        const float* p0 = p.part + size_t(bh + c_first) * G * kMR;
        const int cols = rows * kLanes;
        const int parts = kThreads / cols > 1 ? kThreads / cols : 1;
        const int sub = lane % kLanes;
        for (int e = tid; e < cols * parts; e += kThreads) {  // whole groups of kLanes lanes come through together
          const uint32_t group = kLanes == 32 ? 0xffffffffu : 0xffffu << (lane & 16);
          const int r = e % cols / kLanes, part = e / cols, d = 4 * sub;
          float M = -INFINITY, L = 0.f;
          float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int c0 = part; c0 < np; c0 += kChunk * parts) {
            float4 v[kChunk];
#pragma unroll
            for (int i = 0; i < kChunk; ++i) {
              const int c = c0 + i * parts;
              v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (c < np) v[i] = __ldcg(reinterpret_cast<const float4*>(p0 + (size_t(c) * G + r) * kMR + d));
            }
            const int c = c0 + sub * parts;
            float2 ml = make_float2(-INFINITY, 0.f);
            if (sub < kChunk && c < np) ml = __ldcg(reinterpret_cast<const float2*>(p0 + (size_t(c) * G + r) * kMR + D));
            float m = fmaxf(M, ml.x);
#pragma unroll
            for (int o = 1; o < kLanes; o <<= 1) m = fmaxf(m, __shfl_xor_sync(group, m, o));
            const float old = factor(M, m), f = factor(ml.x, m);
            float l = f * ml.y;
#pragma unroll
            for (int o = 1; o < kLanes; o <<= 1) l += __shfl_xor_sync(group, l, o);
            M = m;
            L = fmaf(L, old, l);
            A.x *= old, A.y *= old, A.z *= old, A.w *= old;
#pragma unroll
            for (int i = 0; i < kChunk; ++i) {
              const float fi = __shfl_sync(group, f, i, kLanes);
              A.x = fmaf(fi, v[i].x, A.x), A.y = fmaf(fi, v[i].y, A.y);
              A.z = fmaf(fi, v[i].z, A.z), A.w = fmaf(fi, v[i].w, A.w);
            }
          }
          if (parts == 1) {
            store_out(out + r * D + d, A, L);
          } else {
            float* j = join + e * 8;
            *reinterpret_cast<float4*>(j) = A;
            *reinterpret_cast<float2*>(j + 4) = make_float2(M, L);
          }
        }
        if (parts > 1) {
          __syncthreads();
          for (int e = tid; e < cols; e += kThreads) {
            const int r = e / (D / 4), d = 4 * (e % (D / 4));
            float M = -INFINITY, L = 0.f;
            float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int c = 0; c < parts; ++c) M = fmaxf(M, join[(c * cols + e) * 8 + 4]);
            for (int c = 0; c < parts; ++c) {
              const float* j = join + (c * cols + e) * 8;
              add_state(A, L, factor(j[4], M), *reinterpret_cast<const float4*>(j), j[5]);
            }
            store_out(out + r * D + d, A, L);
          }
        }
      }
    }
    __syncthreads();  // merge rows free for the next head
  }
  // after a wait that gave up (the results are lost, the counters came out right): leave only once every
  // copy has landed, or never came
  if (*gave_up && lane == 0) {
    for (int i = 0; i < R; ++i) mbar_wait(&full[i], i >= slot ? ph : ph ^ 1u);
  }
}

// More than 8 query heads on a KV head are worked on as two heads: the records' codes are copied and
// unpacked twice (the second time from L2, as a rule), which costs less than two tiles of accumulators in
// one warp, whose registers leave 8 warps on an SM (26 us against 22 with 16 query heads, 141K tokens).
int head_halves(int group) { return group > 8 ? 1 : 0; }

// One place for the counters whatever the number of heads: calls of different sizes may take turns in one
// workspace without one's partial results lying where another counts.
constexpr size_t kCounterBytes = 2 * kMaxBH * 4;

size_t workspace_need(int64_t kv_heads, int group, int D, int sms) {
  const int halves = head_halves(group), G = (group + halves) >> halves;
  const int64_t BH = kv_heads << halves;
  return kCounterBytes + size_t(BH + sms * (kSmWarps / 4)) * G * (D + 4) * 4 + 256;
}

// What an SM has for its CTAs, each of which costs kCtaSmem more than it asks for.
constexpr size_t kSmSmem = 228 * 1024, kCtaSmem = 1024;

struct DecodeLaunch {
  Kv4DecodeParams p;
  cudaStream_t stream;
  int sms, status;
  template <int D, int NG>
  size_t smem_of(int warps) const {
    return fixed_smem(warps, p.BH, p.G, D) + size_t(warps) * kSlots * kNB * Kv4<D, NG>::kRec;
  }
  // CTAs that are on an SM together.  Beside the ring and the merge rows, which let kSmWarps warps in, a CTA
  // holds the line of all heads (8 bytes each), so that from 1800 to 5000 heads up, by D, group and G, three CTAs
  // of 4 warps do not fit, later two of 6 neither.
  template <int D, int NG>
  int resident(int warps) const {
    return int(std::min(size_t(kSmWarps / warps), kSmSmem / (smem_of<D, NG>(warps) + kCtaSmem)));
  }
  template <int D, int NG, int kPack, int kWarps>
  void launch() {
    const int ctas = resident<D, NG>(kWarps);  // a segment for each, all in one wave
    const auto kernel = kv4_decode_kernel<D, NG, kPack, kWarps>;
    const size_t smem = smem_of<D, NG>(kWarps);
    p.slots = kSlots;
    static bool attr_set[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 64 || !attr_set[dev]) {
      if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) != cudaSuccess) {
        status = WGKV_ECUDA;
        return;
      }
      if (dev < 64) attr_set[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(sms * ctas);
    cfg.blockDim = dim3(32 * kWarps);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // set-up overlaps the launch before
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    status = cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? WGKV_OK : WGKV_ECUDA;
  }
  template <int D, int NG, int kPack>
  void warps() {
    if constexpr (kPack == 1)
      if (p.BH < kFewHeads) return launch<D, NG, kPack, 12>();
    // the form for many heads, unless their line leaves fewer of its warps on an SM than of the other's (4096 heads
    // of 200 tokens: 115 us with three CTAs of 4 warps asked for, of which two fit, 70 us with two of 6; 8 rows a
    // head of 100 tokens, groups of 32, where only two CTAs of 4 or one of 6 fit: 113 us with three asked for, 78
    // with two, 112 with one of 12; 8192 such heads of 100 tokens: 248 us with three, 204 with one of 6)
    if (p.BH >= kManyHeads && 4 * resident<D, NG>(4) >= 6 * resident<D, NG>(6)) return launch<D, NG, kPack, 4>();
    launch<D, NG, kPack, 6>();
  }
  template <int D, int NG>
  void run() {
    if (p.G <= 4) warps<D, NG, 2>();
    else warps<D, NG, 1>();
  }
};

}  // namespace
}  // namespace wgkv

using namespace wgkv;

extern "C" size_t wgkv_paged_decode_kv4_workspace_size(int batch, int num_q_heads, int num_kv_heads, int head_dim) {
  if (batch <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || head_dim <= 0) return 0;
  const int sms = device_sms();
  return workspace_need(int64_t(batch) * num_kv_heads, num_q_heads / num_kv_heads, head_dim, sms > 0 ? sms : 148);
}

extern "C" int wgkv_paged_decode_kv4(const uint16_t* q, const uint8_t* cache, int64_t num_pages, int page_size,
                                     int group, const int32_t* cache_seqlens, const int32_t* block_table,
                                     int64_t table_stride, int table_width, int batch, int num_q_heads,
                                     int num_kv_heads, int head_dim, float softmax_scale, uint16_t* out,
                                     void* workspace, size_t workspace_bytes, int* err, void* stream) {
  if (!q || !cache || !cache_seqlens || !block_table || !out || !workspace || !kv4_supported(head_dim, group))
    return WGKV_EINVAL;
  if (batch <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads ||
      num_q_heads / num_kv_heads > kMaxG || int64_t(batch) * num_kv_heads > kMaxBH)
    return WGKV_EINVAL;
  if (num_pages <= 0 || page_size <= 0 || page_size % 16 || table_width <= 0 || table_stride < table_width ||
      (int64_t(batch) * num_kv_heads << head_halves(num_q_heads / num_kv_heads)) * table_width * (page_size / 16) >=
          (int64_t(1) << 29) ||
      int64_t(table_width) * page_size >= (int64_t(1) << 31) || num_pages * (page_size / 16) >= (int64_t(1) << 31) ||
      (reinterpret_cast<uintptr_t>(cache) & 15) || (reinterpret_cast<uintptr_t>(q) & 15) ||
      (reinterpret_cast<uintptr_t>(out) & 15) || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return WGKV_EINVAL;
  if (workspace_bytes < wgkv_paged_decode_kv4_workspace_size(batch, num_q_heads, num_kv_heads, head_dim))
    return WGKV_ENOSPC;
  const int group_heads = num_q_heads / num_kv_heads, halves = head_halves(group_heads);
  DecodeLaunch a = {};
  a.p.c = {const_cast<uint8_t*>(cache), num_pages, page_size, block_table, table_stride, table_width, err};
  a.p.q = q;
  a.p.out = out;
  a.p.seqlens = cache_seqlens;
  a.p.group = group_heads;
  a.p.halves = halves;
  a.p.BH = (batch * num_kv_heads) << halves;
  a.p.G = (group_heads + halves) >> halves;
  a.p.scale_log2 = softmax_scale * 1.4426950408889634f;
  a.p.counters = reinterpret_cast<int*>(workspace);
  a.p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kCounterBytes);
  a.stream = as_stream(stream);
  a.sms = device_sms();
  if (a.sms <= 0) return WGKV_ECUDA;
  kv4_dispatch(head_dim, group, a);
  return a.status;
}
