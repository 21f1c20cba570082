// What the kernels of decode attention over the paged KV cache share (paged_decode.cu, paged_decode_tc.cu): the split of
// the work over CTAs, and the merge of the pieces that the split cuts units into.
#pragma once

#include <algorithm>
#include <atomic>

#include "paged.cuh"
#include "tc.cuh"

namespace fpx {

struct PagedDecodeParams {
  PageView pv;
  int *error;  // the word of waits that gave up, or null
  const __nv_bfloat16 *q;
  int64_t q_sb, q_sl, q_sh;
  __nv_bfloat16 *out;
  int64_t o_sb, o_sl, o_sh;
  float *lse;  // [B][Lq][H] or null
  int B, Lq, H, Hkv, group, blocks;  // blocks: row blocks of 8 NT (query row, head of the group) pairs
  float scale_log2;
  int ctas, min_steps;
  bool whole;      // a CTA a unit, no merge
  int *prefix;     // [B * blocks + 1] steps of all heads before an item (b, row block), with more than 32 items
  float *part_o;   // [ctas + units][8 NT][d]
  float *part_ml;  // [ctas + units][8 NT][2]
};

// The running reference (log2) lies kLift below the logit that set it, and follows when one passes that by kRaise, so
// probabilities are at most 2^(kLift + kRaise). int4 pages: fp16 probabilities, and their products with scales below 2, then
// stay within fp16's range; a token whose weight is 2^-20 of the largest, more than which a million such tokens do not make up for,
// keeps its scale's bits down to 2^-14, fp16's smallest normal number as a scale too. Without the lift u r vanished below
// 2^-25 while the sum of weights kept the token: 131072 tokens 12 nats below one lost 5 % of a group 256 times smaller than the row's largest. bf16
// pages: probabilities are two bf16 terms, which need none.
template <int FMT>
constexpr float kLift = FMT == FPX_PAGES_INT4 ? 10.f : 0.f;
template <int FMT>
constexpr float kRaise = FMT == FPX_PAGES_INT4 ? 4.f : 8.f;
constexpr float kLowest = -3e38f;  // reference before any logit: below all of them, and finite
// Sums of weights stand 2^kSumLift up: against a reference that a value row's exponent e has lifted, a weight lies between 2^(kLift - 125) and
// 2^(kLift + kRaise + 60), and with that factor 2^24 of the largest still are a float, and what vanishes below 2^-126 is a 2^35th of the smallest.
// A weight is u 2^-e, while u < 2^-126 is zero. Where no row's exponent has moved the reference by more than 15, that loses less than a
// 2^50th of the sum. Once one has (is_far), the weights are exponentials of their own: values of 2^60 beside values of
// 2^-60. That code runs where the reference moves, and only costs calls without such values its place there: 14.5 -> 14.8 us for 32641 tokens,
// 65.2 -> 65.5 for a ragged batch of 32.
constexpr float kSumLift = 24.f, kSumUnit = 0x1p24f;

// Keys that row block rb of sequence b needs: all up to its last row's position.
template <int NT>
FPX_INLINE int item_keys(const PagedDecodeParams &p, int start, int count, int rb) {
  const int first = rb * 8 * NT;
  if (first >= count * p.group) return 0;
  const int last = min(count * p.group, first + 8 * NT) - 1;
  const int64_t keys = (int64_t)start + last / p.group + 1;
  if (keys > p.pv.capacity()) {
    p.pv.fail();
    return p.pv.capacity();
  }
  return (int)keys;
}
// A step is the GS granules of one ring stage.
template <int GS>
FPX_INLINE int steps_of(int keys) { return (int)(((unsigned)keys + GS * kGranule - 1) / (GS * kGranule)); }
// What a unit counts in the partition: its steps and, in front of them, what beginning a unit costs a CTA
// (queries, first copies, merge) in steps. 28 columns of 4 x 65536 tokens in steps of 128: 31.1 us with one, 30.4 with two,
// 27.9 with four and six, 29.0 with eight.
constexpr int kPad = 4;
FPX_INLINE int padded(int steps) { return steps ? steps + kPad : 0; }

// What item i (sequence, row block) counts in the partition, all heads together.
template <int NT, int GS>
FPX_INLINE int item_steps(const PagedDecodeParams &p, int i) {
  const int b = i / p.blocks;
  int start, count;
  p.pv.rows(b, p.Lq, start, count);
  return padded(steps_of<GS>(item_keys<NT>(p, start, count, i - b * p.blocks))) * p.Hkv;
}
// Up to 32 items: lane i's steps before its item and of it, and all of them. Every warp does it for itself.
template <int NT, int GS>
FPX_INLINE void lane_items(const PagedDecodeParams &p, int items, int lane, int &before, int &mine, int &total) {
  mine = lane < items ? item_steps<NT, GS>(p, lane) : 0;
  before = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += x;
  }
  total = __shfl_sync(0xffffffffu, before, 31);
  before -= mine;
}

template <int W>
struct Scan {
  int sum[W], item, base;
};

// A CTA's run of the steps, all units' end to end, as the parts of units that it consists of. Uniform over the CTA.
template <int NT, int GS>
struct Walk {
  int lo, hi, item, base;  // lo: where the next part begins; base: where item does
  int b, rb, kvh, start, rows, seen, n_steps, g0, g1;  // the part: steps g0 .. g1 - 1 of the unit's n_steps

  // Finds the run, and the item that it starts in; false: there is none. Leaves the items' sums for the merge.
  template <int W>
  FPX_INLINE bool begin(const PagedDecodeParams &p, Scan<W> &sh, int tid) {
    constexpr int kThreads = 32 * W;
    const int warp = tid >> 5, lane = tid & 31, items = p.B * p.blocks;
    lo = hi = item = base = 0;
    auto run = [&](int total) {
      const int per = max(p.min_steps, (total + p.ctas - 1) / p.ctas);
      lo = (int)min((int64_t)blockIdx.x * per, (int64_t)total);
      hi = min(total, lo + per);
      return lo < hi;
    };
    if (p.whole) {
      item = blockIdx.x / p.Hkv;
      return true;
    }
    if (items <= 32) {
      int before, mine, total;
      lane_items<NT, GS>(p, items, lane, before, mine, total);
      if (!run(total)) return false;
      item = __ffs(__ballot_sync(0xffffffffu, before <= lo && lo < before + mine)) - 1;
      base = __shfl_sync(0xffffffffu, before, item);
      return true;
    }
    const int chunk = (items + kThreads - 1) / kThreads;
    const int i0 = min(items, tid * chunk), i1 = min(items, i0 + chunk);
    int mine = 0;
    for (int i = i0; i < i1; ++i) mine += item_steps<NT, GS>(p, i);
    int before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += x;
    }
    if (lane == 31) sh.sum[warp] = before;
    before -= mine;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w < warp) before += sh.sum[w];
      total += sh.sum[w];
    }
    if (blockIdx.x == 0) {  // for the merge
      int at = before;
      for (int i = i0; i < i1; ++i) {
        p.prefix[i] = at;
        at += chunk == 1 ? mine : item_steps<NT, GS>(p, i);
      }
      if (tid == 0) p.prefix[items] = total;
    }
    if (!run(total)) return false;
    if (before <= lo && lo < before + mine) {
      int at = before;
      for (int i = i0; i < i1; ++i) {
        const int n = chunk == 1 ? mine : item_steps<NT, GS>(p, i);
        if (lo < at + n) {
          sh.item = i;
          sh.base = at;
          break;
        }
        at += n;
      }
    }
    __syncthreads();
    item = sh.item;
    base = sh.base;
    return true;
  }
  FPX_INLINE void read_item(const PagedDecodeParams &p) {
    b = item / p.blocks;
    rb = item - b * p.blocks;
    int count;
    p.pv.rows(b, p.Lq, start, count);
    rows = count * p.group;
    seen = item_keys<NT>(p, start, count, rb);
    n_steps = steps_of<GS>(seen);
  }
  // The next part; false: none is left.
  FPX_INLINE bool find(const PagedDecodeParams &p) {
    while (lo < hi) {
      for (;;) {
        read_item(p);
        if (lo - base < padded(n_steps) * p.Hkv) break;
        base += padded(n_steps) * p.Hkv;
        ++item;
      }
      kvh = (lo - base) / (n_steps + kPad);
      const int first = base + kvh * (n_steps + kPad) + kPad;  // the unit's first step
      g0 = max(0, lo - first);
      g1 = min(n_steps, hi - first);
      lo = first + max(g1, 0);  // hi, or the unit's end
      if (g1 > g0) return true;
    }
    return false;
  }
  FPX_INLINE void whole(const PagedDecodeParams &p) {
    read_item(p);
    kvh = blockIdx.x - item * p.Hkv;
    g0 = 0;
    g1 = n_steps;
  }
};

FPX_INLINE uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
FPX_INLINE uint32_t hmul2u(uint32_t a, uint32_t b) {
  __half2 r = __hmul2(*reinterpret_cast<__half2 *>(&a), *reinterpret_cast<__half2 *>(&b));
  return *reinterpret_cast<uint32_t *>(&r);
}
FPX_INLINE uint32_t hsub2u(uint32_t a, uint32_t b) {
  __half2 r = __hsub2(*reinterpret_cast<__half2 *>(&a), *reinterpret_cast<__half2 *>(&b));
  return *reinterpret_cast<uint32_t *>(&r);
}
FPX_INLINE uint32_t hfma2u(uint32_t a, uint32_t b, uint32_t c) {
  __half2 r = __hfma2(*reinterpret_cast<__half2 *>(&a), *reinterpret_cast<__half2 *>(&b), *reinterpret_cast<__half2 *>(&c));
  return *reinterpret_cast<uint32_t *>(&r);
}
FPX_INLINE uint32_t pack_f16(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t *>(&v);
}
// From products of codes, n 2^-24 of them, and a query times 2^up to log2 units: scale_log2 2^(24 - up). A query above 2^116 may take
// it past a float, and then picks one key whatever its logits' size: there it ends at 2^124, which leaves the products room.
FPX_INLINE float logit_factor(float scale_log2, int up) {
  const int f = 24 - up;
  const float x = scale_log2 * __uint_as_float((uint32_t)(127 + min(f, 127)) << 23);
  return f > 127 ? fminf(fmaxf(x * __uint_as_float((uint32_t)f << 23), -0x1p124f), 0x1p124f) : x;
}
// Of a key's 2^(kSumLift - e): whether e passes 15, and its log2.
FPX_INLINE bool is_far(float w) { return w < kSumUnit / 0x1p15f; }
FPX_INLINE float log2_of(float w) { return (float)((int)(__float_as_uint(w) >> 23) - 127); }
// out = o / l and the log-sum of a row, from sums relative to reference m.
FPX_INLINE float inverse_sum(float l) { return l == 0.f ? 0.f : kSumUnit / l; }
FPX_INLINE float log_sum(float m, float l) { return l == 0.f ? -INFINITY : (m - kSumLift) * kLn2 + logf(l); }
// Loads from a shared-memory address (the granules arrive by bulk copies: ordered by the barrier's wait).
FPX_INLINE uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
FPX_INLINE uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
FPX_INLINE uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
FPX_INLINE uint32_t lds16(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
FPX_INLINE void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// What the merge launches know of a unit: its pieces lie in slots slot .. slot + pieces - 1 (one piece: its CTA has
// finished it; none: no row of it sees anything).
//
// With up to 32 items they work it out from the lengths, before they wait for the main launch (whose CTAs have all waited for
// what came before them by then, so the lengths are there); otherwise from the sums that it left, after.
struct Pieces {
  int b, rb, kvh, rows, pieces;
  int64_t slot;
  template <int NT, int GS>
  FPX_INLINE void find(const PagedDecodeParams &p, int unit, int lane) {
    const int items = p.B * p.blocks, item = unit / p.Hkv;
    kvh = unit - item * p.Hkv;
    b = item / p.blocks;
    rb = item - b * p.blocks;
    int base, n, total;
    if (items <= 32) {
      int before, mine;
      lane_items<NT, GS>(p, items, lane, before, mine, total);
      base = __shfl_sync(0xffffffffu, before, item);
      n = __shfl_sync(0xffffffffu, mine, item) / p.Hkv;
      asm volatile("griddepcontrol.wait;" ::: "memory");
    } else {
      asm volatile("griddepcontrol.wait;" ::: "memory");
      base = p.prefix[item];
      n = (p.prefix[item + 1] - base) / p.Hkv;
      total = p.prefix[items];
    }
    int start, count;
    p.pv.rows(b, p.Lq, start, count);
    rows = count * p.group;
    const int per = max(p.min_steps, (total + p.ctas - 1) / p.ctas);
    const int first = base + kvh * n, c0 = (first + kPad) / per, c1 = (first + n - 1) / per;  // padding, then steps
    pieces = n ? c1 - c0 + 1 : 0;
    slot = c0 + (int64_t)item * p.Hkv + kvh;
  }
};

// Merges the pieces of one (unit, row), where rows are few and pieces many: D / 4 threads a piece, kPieces of them at a
// time, kAhead loads in flight before the weights are known. Rows that see nothing (padding, inactive sequences)
// become zero here.
template <int D, int NT, int GS>
__global__ void __launch_bounds__(512) paged_merge_pieces_kernel(const __grid_constant__ PagedDecodeParams p) {
  constexpr int kThreads = 512, kPieces = kThreads / (D / 4), kRows = 8 * NT, kAhead = 10;
  const int r = blockIdx.y, tid = threadIdx.x, piece = tid / (D / 4), d = 4 * (tid % (D / 4));
  __shared__ float red[kThreads / 32];
  __shared__ __align__(16) float part[kPieces][D];
  __shared__ float weight[kThreads];
  Pieces u{};
  u.find<NT, GS>(p, blockIdx.x, tid & 31);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int rr = u.rb * kRows + r, row = rr / p.group, h = u.kvh * p.group + rr % p.group;
  if (rr >= p.Lq * p.group) return;
  __nv_bfloat16 *out = p.out + u.b * p.o_sb + row * p.o_sl + h * p.o_sh;
  float *lse = p.lse ? p.lse + ((int64_t)u.b * p.Lq + row) * p.H + h : nullptr;
  if (rr >= u.rows || u.pieces == 0) {
    for (int i = tid; i < D; i += kThreads) out[i] = __float2bfloat16_rn(0.f);
    if (lse && tid == 0) *lse = -INFINITY;
    return;
  }
  if (u.pieces == 1) return;
  const float *ml = p.part_ml + 2 * (u.slot * kRows + r), *po = p.part_o + (u.slot * kRows + r) * D + d;
  float m = kLowest, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < u.pieces; i0 += kThreads) {
    const int here = min(u.pieces - i0, kThreads);
    float2 mine = make_float2(kLowest, 0.f);
    if (tid < here) mine = *reinterpret_cast<const float2 *>(ml + 2 * (int64_t)(i0 + tid) * kRows);
    float4 x[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = piece + k * kPieces;
      x[k] = i < here ? *reinterpret_cast<const float4 *>(po + (int64_t)(i0 + i) * kRows * D) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const float top = fmaxf(m, block_max<kThreads>(mine.x, red));  // NaN stays out of m, and in l
    // factors by halves: the whole of one may lie below 2^-126 and its product with a sum above
    const float half_keep = tc::ex2(0.5f * (m - top)), keep = half_keep * half_keep;
    m = top;
    const float half = tid < here ? tc::ex2(0.5f * (mine.x - m)) : 0.f;
    weight[tid] = half * half;
    l = l * half_keep * half_keep + mine.y * half * half;
    o.x *= keep; o.y *= keep; o.z *= keep; o.w *= keep;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = piece + k * kPieces;
      const float w = i < here ? weight[i] : 0.f;
      o.x = fmaf(x[k].x, w, o.x); o.y = fmaf(x[k].y, w, o.y); o.z = fmaf(x[k].z, w, o.z); o.w = fmaf(x[k].w, w, o.w);
    }
#pragma unroll 4
    for (int i = piece + kAhead * kPieces; i < here; i += kPieces) {
      const float4 v = *reinterpret_cast<const float4 *>(po + (int64_t)(i0 + i) * kRows * D);
      const float w = weight[i];
      o.x = fmaf(v.x, w, o.x); o.y = fmaf(v.y, w, o.y); o.z = fmaf(v.z, w, o.z); o.w = fmaf(v.w, w, o.w);
    }
    __syncthreads();
  }
  *reinterpret_cast<float4 *>(&part[piece][d]) = o;
  l = block_sum<kThreads>(l, red);  // its barriers publish part
  const float inv = inverse_sum(l);
  for (int i = tid; i < D; i += kThreads) {
    float x = 0.f;
#pragma unroll
    for (int k = 0; k < kPieces; ++k) x += part[k][i];
    out[i] = __float2bfloat16_rn(x * inv);
  }
  if (lse && tid == 0) *lse = log_sum(m, l);
}

// The same where units are many and pieces few: a warp a row, a block eight or sixteen rows of a unit, D / 32 dims a lane.
template <int NT>
constexpr int kMergeRows = NT == 1 ? 8 : 16;
template <int D, int NT, int GS>
__global__ void __launch_bounds__(32 * kMergeRows<NT>) paged_merge_rows_kernel(const __grid_constant__ PagedDecodeParams p) {
  constexpr int kRows = 8 * NT;
  const int r = blockIdx.y * kMergeRows<NT> + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  Pieces u{};
  u.find<NT, GS>(p, blockIdx.x, lane);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int rr = u.rb * kRows + r, row = rr / p.group, h = u.kvh * p.group + rr % p.group;
  const bool sees = rr < u.rows && u.pieces > 0;
  if (rr >= p.Lq * p.group || (sees && u.pieces == 1)) return;
  float m = kLowest, l = 0.f;
  float4 o[D / 128] = {};
  if (sees) {
    const float *ml = p.part_ml + 2 * (u.slot * kRows + r), *po = p.part_o + (u.slot * kRows + r) * D + 4 * lane;
    constexpr int kAhead = 8;  // pieces whose loads do not wait for the weights
    for (int i0 = 0; i0 < u.pieces; i0 += 32) {
      const int here = min(u.pieces - i0, 32);
      float2 mine = make_float2(kLowest, 0.f);
      if (lane < here) mine = *reinterpret_cast<const float2 *>(ml + 2 * (int64_t)(i0 + lane) * kRows);
      float4 x[kAhead][D / 128];
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
#pragma unroll
        for (int J = 0; J < D / 128; ++J)
          x[k][J] = k < here ? *reinterpret_cast<const float4 *>(po + (int64_t)(i0 + k) * kRows * D + 128 * J)
                             : make_float4(0.f, 0.f, 0.f, 0.f);
      const float top = fmaxf(m, warp_max(mine.x)), half_keep = tc::ex2(0.5f * (m - top)), keep = half_keep * half_keep;
      m = top;
      const float half = lane < here ? tc::ex2(0.5f * (mine.x - m)) : 0.f, s = half * half;
      l = l * half_keep * half_keep + mine.y * half * half;
#pragma unroll
      for (int J = 0; J < D / 128; ++J) {
        o[J].x *= keep; o[J].y *= keep; o[J].z *= keep; o[J].w *= keep;
      }
      auto add = [&](float w, const float4 (&v)[D / 128]) {
#pragma unroll
        for (int J = 0; J < D / 128; ++J) {
          o[J].x = fmaf(v[J].x, w, o[J].x); o[J].y = fmaf(v[J].y, w, o[J].y);
          o[J].z = fmaf(v[J].z, w, o[J].z); o[J].w = fmaf(v[J].w, w, o[J].w);
        }
      };
#pragma unroll
      for (int k = 0; k < kAhead; ++k) add(__shfl_sync(0xffffffffu, s, k), x[k]);
#pragma unroll 4
      for (int i = kAhead; i < here; ++i) {
        float4 v[D / 128];
#pragma unroll
        for (int J = 0; J < D / 128; ++J) v[J] = *reinterpret_cast<const float4 *>(po + (int64_t)(i0 + i) * kRows * D + 128 * J);
        add(__shfl_sync(0xffffffffu, s, i), v);
      }
    }
    l = warp_sum(l);
  }
  const float inv = inverse_sum(l);
  __nv_bfloat16 *out = p.out + u.b * p.o_sb + row * p.o_sl + h * p.o_sh + 4 * lane;
#pragma unroll
  for (int J = 0; J < D / 128; ++J) {
    const float x[4] = {o[J].x * inv, o[J].y * inv, o[J].z * inv, o[J].w * inv};
#pragma unroll
    for (int e = 0; e < 4; ++e) out[128 * J + e] = __float2bfloat16_rn(x[e]);
  }
  if (p.lse && lane == 0) p.lse[((int64_t)u.b * p.Lq + row) * p.H + h] = log_sum(m, l);
}

// ---- host -----------------------------------------------------------------------------------

struct DecodeLayout {
  int nt, blocks, ctas, rows;
  size_t prefix, ml, bytes;
  int64_t units;
};

// Launches the main kernel, as a dependent of what came before it, and the merge after it unless a CTA takes whole units.
template <int D, int NT, int GS, typename Kernel>
static int launch_decode(Kernel kernel, std::atomic<uint64_t> &set, int threads, int smem, int min_steps, PagedDecodeParams &p,
                         const DecodeLayout &w, cudaStream_t stream) {
  // The kernel's shared-memory limit is a setting of the device: once for each.
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return FPX_ERR_CUDA;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (!(set.load(std::memory_order_relaxed) & bit) || !bit) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return FPX_ERR_CUDA;
    set.fetch_or(bit, std::memory_order_relaxed);
  }
  p.min_steps = min_steps;
  // No more CTAs than the table could keep busy.
  const int64_t longest = ((int64_t)p.pv.max_pages << p.pv.page_shift) / GS + 1;  // steps
  const int64_t busy = w.units * (longest + kPad) / p.min_steps + 1;
  p.ctas = (int)(p.whole ? w.units : std::min<int64_t>(w.ctas, busy));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p.ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, p) != cudaSuccess) return FPX_ERR_CUDA;
  if (p.whole) return FPX_OK;
  cfg.dynamicSmemBytes = 0;
  // Few rows have many pieces each, many rows few: a block a row reads them all at once (one sequence of 131072
  // tokens: 7.0 us with a loop over them, 2.5 with this), a warp a row leaves room for more rows (32 sequences of up
  // to 32768: 20 us with a block a row, 5 with this).
  const bool many = w.units * w.rows > 2 * kSms;
  cfg.gridDim = many ? dim3((unsigned)w.units, w.rows / kMergeRows<NT>) : dim3((unsigned)w.units, w.rows);
  cfg.blockDim = dim3(many ? 32 * kMergeRows<NT> : 512);
  const auto merge = many ? paged_merge_rows_kernel<D, NT, GS> : paged_merge_pieces_kernel<D, NT, GS>;
  if (cudaLaunchKernelEx(&cfg, merge, p) != cudaSuccess) return FPX_ERR_CUDA;
  return FPX_OK;
}

// int4 pages, row blocks of 32 or 64 (paged_decode_tc.cu).
int launch_paged_decode_tc(PagedDecodeParams &p, const DecodeLayout &w, int d, cudaStream_t stream);

}  // namespace fpx
