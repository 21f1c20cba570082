// Writing and reading back the paged KV cache: append (rotary embedding on the way, 4-bit
// quantisation for int4 pages) and gather. Page layout: paged.cuh.
#include <algorithm>
#include <atomic>

#include "paged.cuh"
#include "tc.cuh"

namespace fpx {

struct AppendParams {
  PageView pv;
  const __nv_bfloat16 *q, *k, *v;
  int64_t q_sb, q_sl, q_sh, k_sb, k_sl, k_sh, v_sb, v_sl, v_sh;
  __nv_bfloat16 *q_out, *k_out;
  int64_t qo_sb, qo_sl, qo_sh, ko_sb, ko_sl, ko_sh;
  const float *rope;  // [rope_len][rotary]: cosines, then sines; null: no rotation
  int rope_len, rotary;
  int B, L, H, Hkv;   // H = 0: keys and values alone
  int store_rows;     // rows for the pages of a warp, kStoreRows or half of them
  bool zero_padding, q_wide, kv_wide;  // wide: q and q_out, or k, v and k_out, are 16-byte aligned rows
};

// A warp's share of a head row: lane holds dims 128 J + 4 lane .. + 3, as two packed words.
template <int D>
struct HeadRow {
  uint2 w[D / 128];
};
template <int D>
FPX_INLINE HeadRow<D> load_row(const __nv_bfloat16 *p, int lane) {
  HeadRow<D> r;
#pragma unroll
  for (int J = 0; J < D / 128; ++J) r.w[J] = *reinterpret_cast<const uint2 *>(p + 128 * J + 4 * lane);
  return r;
}
template <int D>
FPX_INLINE void unpack_row(const HeadRow<D> &r, float (&x)[D / 128][4]) {
#pragma unroll
  for (int J = 0; J < D / 128; ++J) {
    x[J][0] = __uint_as_float(r.w[J].x << 16);
    x[J][1] = __uint_as_float(r.w[J].x & 0xffff0000u);
    x[J][2] = __uint_as_float(r.w[J].y << 16);
    x[J][3] = __uint_as_float(r.w[J].y & 0xffff0000u);
  }
}
template <int D>
FPX_INLINE void store_row(__nv_bfloat16 *p, const float (&x)[D / 128][4], int lane) {
#pragma unroll
  for (int J = 0; J < D / 128; ++J)
    *reinterpret_cast<uint2 *>(p + 128 * J + 4 * lane) = make_uint2(pack_bf16(x[J][0], x[J][1]), pack_bf16(x[J][2], x[J][3]));
}

// Cosines and sines of this lane's dims (zero where a dim does not rotate), and the sign of
// the partner's product: dims below rotary / 2 take x c - y s, those above x c + y s.
template <int D>
struct Turn {
  float c[D / 128][4], s[D / 128][4];
};
template <int D>
FPX_INLINE Turn<D> load_turn(const float *row, int rotary, int lane) {
  Turn<D> t;
  const int half = rotary >> 1;
#pragma unroll
  for (int J = 0; J < D / 128; ++J) {
    const int d = 128 * J + 4 * lane;
    if (d >= rotary) continue;
    const int i = d < half ? d : d - half;
    const float4 c = *reinterpret_cast<const float4 *>(row + i), s = *reinterpret_cast<const float4 *>(row + half + i);
    const float sg = d < half ? -1.f : 1.f;
    t.c[J][0] = c.x; t.c[J][1] = c.y; t.c[J][2] = c.z; t.c[J][3] = c.w;
    t.s[J][0] = sg * s.x; t.s[J][1] = sg * s.y; t.s[J][2] = sg * s.z; t.s[J][3] = sg * s.w;
  }
  return t;
}
// Rotates a row: each product and the sum rounded in fp32 (no fused multiply-add), so that the
// result is the formula's in fp32 whatever the compiler contracts. The partner dims (+- rotary / 2, a
// multiple of 4) belong to one other lane; their packed words come by shuffles.
template <int D>
FPX_INLINE void rotate_row(const HeadRow<D> &r, const Turn<D> &t, int rotary, int lane, float (&x)[D / 128][4]) {
  unpack_row<D>(r, x);
  const int half = rotary >> 1;
#pragma unroll
  for (int J = 0; J < D / 128; ++J) {
    const int d = 128 * J + 4 * lane;
    const int other = d < half ? d + half : d - half;  // partner's dim (for d < rotary)
    const int from = (other >> 2) & 31;
    uint2 y;
    y.x = __shfl_sync(0xffffffffu, r.w[0].x, from);
    y.y = __shfl_sync(0xffffffffu, r.w[0].y, from);
    if (D == 256) {
      const uint32_t hx = __shfl_sync(0xffffffffu, r.w[D / 128 - 1].x, from);
      const uint32_t hy = __shfl_sync(0xffffffffu, r.w[D / 128 - 1].y, from);
      if (other >= 128) y = make_uint2(hx, hy);
    }
    if (d < rotary) {
      const float p[4] = {__uint_as_float(y.x << 16), __uint_as_float(y.x & 0xffff0000u), __uint_as_float(y.y << 16),
                          __uint_as_float(y.y & 0xffff0000u)};
#pragma unroll
      for (int e = 0; e < 4; ++e) x[J][e] = __fadd_rn(__fmul_rn(x[J][e], t.c[J][e]), __fmul_rn(p[e], t.s[J][e]));
    }
  }
}

// m / 7 correctly rounded, by the quick division of codes4 where nothing under- or overflows.
FPX_INLINE float seventh(float m) {
  if (!(m > 0x1p-100f && m < 0x1p100f)) return __fdiv_rn(m, 7.f);
  constexpr float kInv = 1.f / 7.f;
  const float q = __fmul_rn(m, kInv);
  return __fmaf_rn(__fmaf_rn(-q, 7.f, m), kInv, q);
}
FPX_INLINE float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// The four codes of x / s, low nibble first.
//
// quick: s is a normal number between 2^-100 and 2^100 whose relative rounding is at most 2^-8, so |x / s| rounds to 7
// at most; `inv` is 1 / s correctly rounded. Then q = x inv, and q + (x - q s) inv is x / s correctly rounded
// (Markstein's theorem on division by a rounded reciprocal; s has no mantissa of ones), at a third of a division's
// instructions. Adding 1.5 * 2^23 + 8 rounds to the nearest even integer and leaves the code in the low bits.
// Otherwise: a scale of zero gives the middle code, 0 * s; so does one that is no number or infinite, whose 0 * s is
// NaN.
FPX_INLINE uint32_t codes4(const float (&x)[4], float s, float inv, bool quick) {
  if (quick) {
    uint32_t n[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float q = __fmul_rn(x[e], inv);
      n[e] = __float_as_uint(__fadd_rn(__fmaf_rn(__fmaf_rn(-q, s, x[e]), inv, q), 12582920.f));
    }
    return ((n[3] * 16 + n[2]) * 16 + n[1]) * 16 + n[0];  // the low 16 bits: 1.5 * 2^23's are zero
  }
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float n = s > 0.f && s < INFINITY ? fminf(fmaxf(rintf(__fdiv_rn(x[e], s)), -7.f), 7.f) : 0.f;
    w |= (uint32_t)((int)n + 8) << (4 * e);
  }
  return w;
}

// A value row's exponent and the factors to and from its scales, from the lane's N groups (a: amax / 7) and the lanes of the row, FIRST,
// 2 FIRST .. < LANES apart. An infinity or a NaN among them means exponent 126, where the scales of other groups below 2^101 are
// zero. Where they all are, it is -60, as for a row of zeros: it joins the logit in attention, and 126 there would take the other
// rows' bits.
template <int N, int FIRST, int LANES>
struct RowExponent {
  int e;
  float up, down;
  FPX_INLINE explicit RowExponent(const float (&a)[N]) {
    float top = a[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = max_nan(top, a[i]);
#pragma unroll
    for (int o = FIRST; o < LANES; o <<= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    e = min(max((int)((__float_as_uint(top) >> 23) & 255u) - 127, -60), 126);
    up = __uint_as_float((uint32_t)(e + 127) << 23);
    down = __uint_as_float((uint32_t)(127 - e) << 23);
    const bool number = e < 126;  // finite ones end at 2^125.2
    if (__any_sync(0xffffffffu, !number)) {
      float most = 0.f;  // of the others
#pragma unroll
      for (int i = 0; i < N; ++i) most = a[i] < INFINITY ? fmaxf(most, a[i]) : most;
#pragma unroll
      for (int o = FIRST; o < LANES; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      if (!number && __half2float(__float2half_rn(most * down)) == 0.f) {
        e = -60;
        up = 0x1p-60f;
        down = 0.f;
      }
    }
  }
};

// One row of K (VALUE false) or V into the granule of token t.
template <int D, bool VALUE>
FPX_INLINE void write_int4(uint8_t *gran, int t, const float (&x)[D / 128][4], int lane) {
  using G = Granule<FPX_PAGES_INT4, D>;
  const int j = lane >> 3;
  float a[D / 128];
#pragma unroll
  for (int J = 0; J < D / 128; ++J) {
    float m = max_nan(max_nan(fabsf(x[J][0]), fabsf(x[J][1])), max_nan(fabsf(x[J][2]), fabsf(x[J][3])));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    a[J] = seventh(m);
  }
  if (VALUE) {
    const RowExponent<D / 128, 8, 32> x2(a);
#pragma unroll
    for (int J = 0; J < D / 128; ++J) {
      const __half r = __float2half_rn(a[J] * x2.down);
      const float s = __half2float(r) * x2.up;
      const uint32_t w = codes4(x[J], s, __frcp_rn(s), s > 0x1p-100f && s < 0x1p100f && __half2float(r) >= 0x1p-14f);
      *reinterpret_cast<uint16_t *>(gran + G::kVCodes + v_chunk(t, J, lane & 7) + 2 * j) = (uint16_t)w;
      if ((lane & 7) == 0)
        *reinterpret_cast<__half *>(gran + G::kVScales + (((t >> 1) * (D / 32) + 4 * J + j) * 2 + (t & 1)) * 2) = r;
    }
    if (lane == 0) *reinterpret_cast<__nv_bfloat16 *>(gran + G::kVExps + 2 * t) = __float2bfloat16_rn((float)x2.e);
  } else {
    const int p = (lane & 7) >> 1;
#pragma unroll
    for (int J = 0; J < D / 128; ++J) {
      const __nv_bfloat16 s = __float2bfloat16_rn(a[J]);
      const float f = __bfloat162float(s);
      const uint32_t w = codes4(x[J], f, __frcp_rn(f), f > 0x1p-100f && f < 0x1p100f);
      *reinterpret_cast<uint16_t *>(gran + t * (D / 2) + J * 64 + (4 * p + j) * 4 + (lane & 1) * 2) = (uint16_t)w;
      if ((lane & 7) == 0) *reinterpret_cast<__nv_bfloat16 *>(gran + G::kKScales + (t * (D / 32) + 4 * J + j) * 2) = s;
    }
  }
}

// bf16 pages: lane's 4 dims are half a 16-byte chunk.
template <int D, bool VALUE>
FPX_INLINE void write_bf16(uint8_t *gran, int t, const float (&x)[D / 128][4], int lane) {
  using G = Granule<FPX_PAGES_BF16, D>;
#pragma unroll
  for (int J = 0; J < D / 128; ++J) {
    const int c = 16 * J + (lane >> 1);
    uint8_t *dst = gran + t * G::kRow + (VALUE ? 2 * D : 0) + ((c ^ (t & 7)) << 4) + ((lane & 1) << 3);
    *reinterpret_cast<uint2 *>(dst) = make_uint2(pack_bf16(x[J][0], x[J][1]), pack_bf16(x[J][2], x[J][3]));
  }
}

// The granule of position pos of sequence b and head kvh, or null with the error word set.
FPX_INLINE uint8_t *granule_of(const PageView &pv, int b, int pos, int kvh, int granule_bytes) {
  if (pos >= pv.capacity()) {
    pv.fail();
    return nullptr;
  }
  const int g = pos >> 4;
  const int page = pv.table[(int64_t)b * pv.table_stride + (g >> pv.page_shift)];
  if ((unsigned)page >= (unsigned)pv.pages) {
    pv.fail();
    return nullptr;
  }
  return pv.pool + (int64_t)page * pv.page_bytes + (int64_t)kvh * pv.head_bytes +
         (int64_t)(g & ((1 << pv.page_shift) - 1)) * granule_bytes;
}

constexpr int kPasses = 8;                                     // of a warp over query heads
constexpr int query_heads(int d) { return kPasses * 32 / (d / 8); }
constexpr int kStoreRows = 8;                                  // rows of [k heads | v heads] of a warp, at most

// Queries of which a part rotates (or nothing): D / 8 lanes a head row. A lane holds four dims and the four that they rotate with (or eight that do not
// rotate), so a rotation stays in the lane; the token's cosines and sines are loaded once for all of the warp's heads.
template <int D>
FPX_INLINE void append_queries_partly(const AppendParams &p, int b, int l, int pos, int h0, bool live, int lane) {
  constexpr int kLanes = D / 8, kRows = 32 / kLanes;
  const int u = lane % kLanes, sub = lane / kLanes, rotary = p.rope ? p.rotary : 0;
  const bool turns = 8 * u < rotary;
  const int d0 = turns ? 4 * u : 8 * u, d1 = turns ? 4 * u + rotary / 2 : 8 * u + 4;
  const __nv_bfloat16 *src = p.q + b * p.q_sb + l * p.q_sl;
  __nv_bfloat16 *dst = p.q_out + b * p.qo_sb + l * p.qo_sl;
  uint2 x[kPasses], y[kPasses];
  if (live) {
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int h = h0 + kRows * i + sub;
      if (h < p.H) {
        x[i] = *reinterpret_cast<const uint2 *>(src + h * p.q_sh + d0);
        y[i] = *reinterpret_cast<const uint2 *>(src + h * p.q_sh + d1);
      }
    }
  }
  float c[4], s[4];
  if (turns && live) {
    const float *row = p.rope + (int64_t)pos * rotary;
    const float4 cv = *reinterpret_cast<const float4 *>(row + 4 * u), sv = *reinterpret_cast<const float4 *>(row + rotary / 2 + 4 * u);
    c[0] = cv.x; c[1] = cv.y; c[2] = cv.z; c[3] = cv.w;
    s[0] = sv.x; s[1] = sv.y; s[2] = sv.z; s[3] = sv.w;
  }
  __syncwarp();  // q_out may be q: a lane stores only after every lane has loaded
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int h = h0 + kRows * i + sub;
    if (h >= p.H) continue;
    uint2 ox = make_uint2(0, 0), oy = ox;
    if (live) {
      ox = x[i];
      oy = y[i];
      if (turns) {  // each product and each sum rounded (no fused multiply-add), as rotate_row
        const float a[4] = {__uint_as_float(ox.x << 16), __uint_as_float(ox.x & 0xffff0000u), __uint_as_float(ox.y << 16),
                            __uint_as_float(ox.y & 0xffff0000u)};
        const float z[4] = {__uint_as_float(oy.x << 16), __uint_as_float(oy.x & 0xffff0000u), __uint_as_float(oy.y << 16),
                            __uint_as_float(oy.y & 0xffff0000u)};
        float m[4], n[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          m[e] = __fsub_rn(__fmul_rn(a[e], c[e]), __fmul_rn(z[e], s[e]));
          n[e] = __fadd_rn(__fmul_rn(z[e], c[e]), __fmul_rn(a[e], s[e]));
        }
        ox = make_uint2(pack_bf16(m[0], m[1]), pack_bf16(m[2], m[3]));
        oy = make_uint2(pack_bf16(n[0], n[1]), pack_bf16(n[2], n[3]));
      }
    }
    *reinterpret_cast<uint2 *>(dst + h * p.qo_sh + d0) = ox;
    *reinterpret_cast<uint2 *>(dst + h * p.qo_sh + d1) = oy;
  }
}

// Eight neighbouring dims; head rows are 8-byte aligned at least.
FPX_INLINE uint4 load8(const __nv_bfloat16 *src, bool wide) {
  if (wide) return *reinterpret_cast<const uint4 *>(src);
  const uint2 lo = *reinterpret_cast<const uint2 *>(src), hi = *reinterpret_cast<const uint2 *>(src + 4);
  return make_uint4(lo.x, lo.y, hi.x, hi.y);
}
FPX_INLINE void store8(__nv_bfloat16 *dst, uint4 v, bool wide) {
  if (wide) {
    *reinterpret_cast<uint4 *>(dst) = v;
  } else {
    *reinterpret_cast<uint2 *>(dst) = make_uint2(v.x, v.y);
    *reinterpret_cast<uint2 *>(dst + 4) = make_uint2(v.z, v.w);
  }
}
FPX_INLINE void unpack8(uint4 w, float (&x)[8]) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = __uint_as_float(v[e] << 16);
    x[2 * e + 1] = __uint_as_float(v[e] & 0xffff0000u);
  }
}
FPX_INLINE uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}
// Cosines and sines of dims 8 u .. + 7, where the whole head rotates; x and its partners half a head away, as
// rotate_row: each product and each sum rounded (no fused multiply-add).
template <int D>
struct WholeTurn {
  float c[8], s[8];
  FPX_INLINE void load(const float *rope, int pos, int u) {
    const float4 *row = reinterpret_cast<const float4 *>(rope + (int64_t)pos * D + 8 * u);
    const float4 v[4] = {row[0], row[1], row[D / 8], row[D / 8 + 1]};
    c[0] = v[0].x; c[1] = v[0].y; c[2] = v[0].z; c[3] = v[0].w; c[4] = v[1].x; c[5] = v[1].y; c[6] = v[1].z; c[7] = v[1].w;
    s[0] = v[2].x; s[1] = v[2].y; s[2] = v[2].z; s[3] = v[2].w; s[4] = v[3].x; s[5] = v[3].y; s[6] = v[3].z; s[7] = v[3].w;
  }
  FPX_INLINE void turn(float (&x)[2][8]) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = x[0][e], z = x[1][e];
      x[0][e] = __fsub_rn(__fmul_rn(a, c[e]), __fmul_rn(z, s[e]));
      x[1][e] = __fadd_rn(__fmul_rn(z, c[e]), __fmul_rn(a, s[e]));
    }
  }
};

// Queries that rotate as a whole: D / 16 lanes a head row, the token's cosines and sines loaded once for the warp's heads.
template <int D>
FPX_INLINE void append_queries(const AppendParams &p, int b, int l, int pos, int h0, bool live, int lane) {
  constexpr int kLanes = D / 16, kRows = 32 / kLanes, kTimes = query_heads(D) / kRows;
  const int u = lane % kLanes, sub = lane / kLanes;
  const __nv_bfloat16 *src = p.q + b * p.q_sb + l * p.q_sl + 8 * u;
  __nv_bfloat16 *dst = p.q_out + b * p.qo_sb + l * p.qo_sl + 8 * u;
  uint4 w[kTimes][2];
#pragma unroll
  for (int i = 0; i < kTimes; ++i) {
    const int h = h0 + kRows * i + sub;
    w[i][0] = w[i][1] = make_uint4(0, 0, 0, 0);
    if (!live || h >= p.H) continue;
    w[i][0] = load8(src + h * p.q_sh, p.q_wide);
    w[i][1] = load8(src + h * p.q_sh + D / 2, p.q_wide);
  }
  WholeTurn<D> turn;
  if (live) turn.load(p.rope, pos, u);
  __syncwarp();  // q_out may be q: a lane stores only after every lane has loaded
#pragma unroll
  for (int i = 0; i < kTimes; ++i) {
    const int h = h0 + kRows * i + sub;
    if (h >= p.H) continue;
    if (live) {
      float x[2][8];
      unpack8(w[i][0], x[0]);
      unpack8(w[i][1], x[1]);
      turn.turn(x);
      w[i][0] = pack8(x[0]);
      w[i][1] = pack8(x[1]);
    }
    store8(dst + h * p.qo_sh, w[i][0], p.q_wide);
    store8(dst + h * p.qo_sh + D / 2, w[i][1], p.q_wide);
  }
}

// Keys and values into their pages, where the whole head or nothing of it rotates: D / 16 lanes a row. A lane holds
// dims 8 u .. + 7 and 8 u + d / 2 .. + 7, which rotate with each other; four lanes hold a group of 32.
template <int FMT, int D>
FPX_INLINE void append_rows(const AppendParams &p, int b, int l, int pos, uint8_t *gran, int r0, int lane) {
  constexpr int kLanes = D / 16, kRows = 32 / kLanes;
  const int u = lane % kLanes, last = min(r0 + p.store_rows, 2 * p.Hkv), t = pos & (kGranule - 1);
  uint4 w[kStoreRows / kRows][2];
#pragma unroll
  for (int i = 0; i < kStoreRows / kRows; ++i) {
    const int r = r0 + kRows * i + lane / kLanes;
    w[i][0] = w[i][1] = make_uint4(0, 0, 0, 0);
    if (r >= last) continue;
    const __nv_bfloat16 *src = r < p.Hkv ? p.k + b * p.k_sb + l * p.k_sl + r * p.k_sh
                                         : p.v + b * p.v_sb + l * p.v_sl + (r - p.Hkv) * p.v_sh;
    w[i][0] = load8(src + 8 * u, p.kv_wide);
    w[i][1] = load8(src + 8 * u + D / 2, p.kv_wide);
  }
  WholeTurn<D> turn;
  if (p.rope && r0 < p.Hkv) turn.load(p.rope, pos, u);
  __syncwarp();  // k_out may be k: a lane stores only after every lane has loaded
#pragma unroll
  for (int i = 0; i < kStoreRows / kRows; ++i) {
    if (r0 + kRows * i >= last) break;
    const int r = r0 + kRows * i + lane / kLanes;
    const bool value = r >= p.Hkv, mine = r < last;
    const int kvh = value ? r - p.Hkv : r;
    float x[2][8];
    unpack8(w[i][0], x[0]);
    unpack8(w[i][1], x[1]);
    if (!value && p.rope) turn.turn(x);
    if (FMT == FPX_PAGES_BF16 || (!value && p.k_out)) {
      w[i][0] = pack8(x[0]);
      w[i][1] = pack8(x[1]);
      if (!value && p.k_out && mine) {
        __nv_bfloat16 *dst = p.k_out + b * p.ko_sb + l * p.ko_sl + kvh * p.ko_sh + 8 * u;
        store8(dst, w[i][0], p.kv_wide);
        store8(dst + D / 2, w[i][1], p.kv_wide);
      }
    }
    uint8_t *page = gran + (int64_t)kvh * p.pv.head_bytes;
    if constexpr (FMT == FPX_PAGES_BF16) {
      if (mine && gran) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<uint4 *>(page + t * Granule<FMT, D>::kRow + (value ? 2 * D : 0) + (((u + h * (D / 16)) ^ (t & 7)) << 4)) =
              w[i][h];
      }
    } else {
      using G = Granule<FPX_PAGES_INT4, D>;
      float a[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float m = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) m = max_nan(m, fabsf(x[h][e]));
        m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 2));
        a[h] = seventh(m);
      }
      const RowExponent<2, 4, kLanes> x2(a);
      if (!mine || !gran) continue;  // no lane of the warp waits for another below
      const int part = u & 3;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int dim = 8 * u + h * (D / 2), J = dim >> 7, j = (dim & 127) >> 5;
        const __half r16 = __float2half_rn(a[h] * x2.down);
        const __nv_bfloat16 b16 = __float2bfloat16_rn(a[h]);
        const float sc = value ? __half2float(r16) * x2.up : __bfloat162float(b16);
        const bool quick = sc > 0x1p-100f && sc < 0x1p100f && (!value || __half2float(r16) >= 0x1p-14f);
        const float inv = __frcp_rn(sc);
        const uint32_t lo = codes4({x[h][0], x[h][1], x[h][2], x[h][3]}, sc, inv, quick);
        const uint32_t hi = codes4({x[h][4], x[h][5], x[h][6], x[h][7]}, sc, inv, quick);
        if (value) {
          *reinterpret_cast<uint16_t *>(page + G::kVCodes + v_chunk(t, J, 2 * part) + 2 * j) = (uint16_t)lo;
          *reinterpret_cast<uint16_t *>(page + G::kVCodes + v_chunk(t, J, 2 * part + 1) + 2 * j) = (uint16_t)hi;
          if (part == 0)
            *reinterpret_cast<__half *>(page + G::kVScales + (((t >> 1) * (D / 32) + 4 * J + j) * 2 + (t & 1)) * 2) = r16;
        } else {
          *reinterpret_cast<uint32_t *>(page + t * (D / 2) + J * 64 + (4 * part + j) * 4) = __byte_perm(lo, hi, 0x5410);
          if (part == 0) *reinterpret_cast<__nv_bfloat16 *>(page + G::kKScales + (t * (D / 32) + 4 * J + j) * 2) = b16;
        }
      }
      if (value && u == 0) *reinterpret_cast<__nv_bfloat16 *>(page + G::kVExps + 2 * t) = __float2bfloat16_rn((float)x2.e);
    }
  }
}

// The same where a part of the head rotates: a warp a row, four dims a lane.
template <int FMT, int D>
FPX_INLINE void append_rows_partly(const AppendParams &p, int b, int l, int pos, uint8_t *gran, int r0, int lane) {
  const int last = min(r0 + p.store_rows, 2 * p.Hkv), t = pos & (kGranule - 1);
  Turn<D> turn{};
  if (r0 < p.Hkv) turn = load_turn<D>(p.rope + (int64_t)pos * p.rotary, p.rotary, lane);
  HeadRow<D> rows[kStoreRows];
#pragma unroll
  for (int i = 0; i < kStoreRows; ++i) {
    const int r = r0 + i;
    if (r >= last) break;
    rows[i] = load_row<D>(r >= p.Hkv ? p.v + b * p.v_sb + l * p.v_sl + (r - p.Hkv) * p.v_sh
                                     : p.k + b * p.k_sb + l * p.k_sl + r * p.k_sh, lane);
  }
  __syncwarp();  // k_out may be k: a lane stores only after every lane has loaded
#pragma unroll
  for (int i = 0; i < kStoreRows; ++i) {
    const int r = r0 + i;
    if (r >= last) break;
    float x[D / 128][4];
    const bool value = r >= p.Hkv;
    const int kvh = value ? r - p.Hkv : r;
    if (value)
      unpack_row<D>(rows[i], x);
    else
      rotate_row<D>(rows[i], turn, p.rotary, lane, x);
    if (!value && p.k_out) store_row<D>(p.k_out + b * p.ko_sb + l * p.ko_sl + kvh * p.ko_sh, x, lane);
    if (!gran) continue;
    uint8_t *page = gran + (int64_t)kvh * p.pv.head_bytes;
    if (FMT == FPX_PAGES_INT4) {
      if (value)
        write_int4<D, true>(page, t, x, lane);
      else
        write_int4<D, false>(page, t, x, lane);
    } else {
      if (value)
        write_bf16<D, true>(page, t, x, lane);
      else
        write_bf16<D, false>(page, t, x, lane);
    }
  }
}

// A warp a token: blocks of the grid's second dim below query_chunks take query_heads(D) query heads each, the others
// store_rows rows for the pages. Six blocks an SM (the registers of one row pass) measured
// 110 us for 32640 tokens of 28 + 2 x 4 heads, five 116.
template <int FMT, int D>
__global__ void __launch_bounds__(128, 6) paged_append_kernel(const __grid_constant__ AppendParams p, int query_chunks) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const uint32_t token = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (token >= (uint32_t)p.B * (uint32_t)p.L) return;
  const int b = (int)(token / (uint32_t)p.L), l = (int)(token - (uint32_t)b * p.L);
  int start, count;
  p.pv.rows(b, p.L, start, count);
  const int64_t pos64 = (int64_t)start + l;
  const bool row = l < count, past = pos64 > 0x7ffffffe || (p.rope && pos64 >= p.rope_len);
  if (row && past) p.pv.fail();
  const bool live = row && !past;
  if (!live && !p.zero_padding) return;
  const int pos = (int)pos64;
  if ((int)blockIdx.y < query_chunks) {
    if (p.rope && p.rotary == D)
      append_queries<D>(p, b, l, pos, blockIdx.y * query_heads(D), live, lane);
    else
      append_queries_partly<D>(p, b, l, pos, blockIdx.y * query_heads(D), live, lane);
    return;
  }
  const int r0 = (blockIdx.y - query_chunks) * p.store_rows;
  if (!live) {
    const float zero[D / 128][4] = {};
    for (int r = r0; r < min(r0 + p.store_rows, p.Hkv) && p.k_out; ++r)
      store_row<D>(p.k_out + b * p.ko_sb + l * p.ko_sl + r * p.ko_sh, zero, lane);
    return;
  }
  uint8_t *gran = granule_of(p.pv, b, pos, 0, Granule<FMT, D>::kBytes);
  if (!p.rope || p.rotary == D)
    append_rows<FMT, D>(p, b, l, pos, gran, r0, lane);
  else
    append_rows_partly<FMT, D>(p, b, l, pos, gran, r0, lane);
}

struct GatherParams {
  PageView pv;
  __nv_bfloat16 *k, *v;
  int64_t k_sb, k_sl, k_sh, v_sb, v_sl, v_sh;
  int B, L, Hkv;
  bool zero_padding, wide;
};

// Rows of one granule that a warp writes: row of token t is first + t. live: bit t: it comes from the page; zero: it
// becomes zero.
struct GatherRows {
  __nv_bfloat16 *k, *v;  // of row `first`, which may lie before the output's first
  int64_t k_sl, v_sl;
  uint32_t live, zero;
  bool wide;  // the output's rows are 16-byte aligned
};
// bf16(n - 8) s of a word of eight codes, correctly rounded (both factors are bf16): codes become 128 + n by an
// and-or of two of them, four dims apart, 136 is taken off exactly, and the products are put back in order.
FPX_INLINE uint4 scaled8(uint32_t w, __nv_bfloat162 s) {
  uint32_t p[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
    const __nv_bfloat162 x = __hmul2(__hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&u), __floats2bfloat162_rn(136.f, 136.f)), s);
    p[i] = *reinterpret_cast<const uint32_t *>(&x);
  }
  return make_uint4(__byte_perm(p[0], p[1], 0x5410), __byte_perm(p[2], p[3], 0x5410), __byte_perm(p[0], p[1], 0x7632),
                    __byte_perm(p[2], p[3], 0x7632));
}

// int4: a lane reads 16 bytes of codes: of keys, its parts of four groups of one token (eight dims each), of values, four dims of four groups
// of a token pair. Quads and eights of lanes write 64 contiguous bytes.
template <int D>
FPX_INLINE void gather_int4(const GatherRows &o, const uint8_t *gran, int lane) {
  using G = Granule<FPX_PAGES_INT4, D>;
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int J = 0; J < D / 128; ++J)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int token = g + 8 * half;
      const bool live = (o.live >> token) & 1;
      if (!live && !((o.zero >> token) & 1)) continue;
      uint4 w = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
      uint2 sc = make_uint2(0, 0);
      if (live) {
        w = *reinterpret_cast<const uint4 *>(gran + token * (D / 2) + 64 * J + 16 * t);
        sc = *reinterpret_cast<const uint2 *>(gran + G::kKScales + token * (D / 16) + 8 * J);
      }
      const uint32_t words[4] = {w.x, w.y, w.z, w.w};
      __nv_bfloat16 *dst = o.k + token * o.k_sl + 128 * J + 8 * t;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t u = j < 2 ? sc.x : sc.y;
        const uint32_t s = __byte_perm(u, u, j & 1 ? 0x3232 : 0x1010);
        store8(dst + 32 * j, scaled8(words[j], *reinterpret_cast<const __nv_bfloat162 *>(&s)), o.wide);
      }
    }
  const int vg = lane & 7;
#pragma unroll
  for (int J = 0; J < D / 128; ++J)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int q = (lane >> 3) + 4 * half;  // token pair
      const uint32_t mine = 3u << (2 * q);
      if (!((o.live | o.zero) & mine)) continue;
      uint4 w = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u), sc = make_uint4(0, 0, 0, 0);
      uint32_t e2 = 0;
      if (o.live & mine) {
        w = *reinterpret_cast<const uint4 *>(gran + G::kVCodes + v_chunk(2 * q, J, vg));
        sc = *reinterpret_cast<const uint4 *>(gran + G::kVScales + q * (D / 8) + 16 * J);
        e2 = *reinterpret_cast<const uint32_t *>(gran + G::kVExps + 4 * q);
      }
      const uint32_t scales[4] = {sc.x, sc.y, sc.z, sc.w};
#pragma unroll
      for (int odd = 0; odd < 2; ++odd) {
        const int token = 2 * q + odd;
        const bool live = (o.live >> token) & 1;
        if (!live && !((o.zero >> token) & 1)) continue;
        const float e = __uint_as_float(odd ? e2 & 0xffff0000u : e2 << 16);
        const float up = __uint_as_float((uint32_t)((int)e + 127) << 23);
        const uint32_t words[2] = {odd ? w.z : w.x, odd ? w.w : w.y};
        __nv_bfloat16 *dst = o.v + token * o.v_sl + 128 * J + 4 * vg;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const __half2 r2 = *reinterpret_cast<const __half2 *>(&scales[j]);
          const float s = live ? __half2float(odd ? __high2half(r2) : __low2half(r2)) * up : 0.f;
          float x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)  // 2^23 + n in the float's bits
            x[i] = live ? (__uint_as_float(((words[j >> 1] >> (16 * (j & 1) + 4 * i)) & 15u) | 0x4b000000u) - 8388616.f) * s : 0.f;
          *reinterpret_cast<uint2 *>(dst + 32 * j) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
        }
      }
    }
}

// bf16: 16-byte chunks, unswizzled.
template <int D>
FPX_INLINE void gather_bf16(const GatherRows &o, const uint8_t *gran, int lane) {
  using G = Granule<FPX_PAGES_BF16, D>;
  constexpr int kChunks = D / 8;  // of K, and of V
  constexpr int kAhead = 8;  // loads in flight
  for (int i0 = lane; i0 < kGranule * 2 * kChunks; i0 += 32 * kAhead) {
    uint4 w[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = i0 + 32 * k, token = i / (2 * kChunks), c = i % kChunks;
      w[k] = make_uint4(0, 0, 0, 0);
      if ((o.live >> token) & 1)
        w[k] = *reinterpret_cast<const uint4 *>(gran + token * G::kRow + ((i / kChunks) & 1 ? 2 * D : 0) + ((c ^ (token & 7)) << 4));
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = i0 + 32 * k, token = i / (2 * kChunks), c = i % kChunks;
      if (((o.live | o.zero) >> token) & 1)
        store8(((i / kChunks) & 1 ? o.v + token * o.v_sl : o.k + token * o.k_sl) + 8 * c, w[k], o.wide);
    }
  }
}

// A warp a granule of one sequence and KV head: its rows are those of the call whose positions lie in it.
template <int FMT, int D>
__global__ void __launch_bounds__(128) paged_gather_kernel(const __grid_constant__ GatherParams p, int granules) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31, kvh = blockIdx.y;
  const int64_t index = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (index >= (int64_t)p.B * granules) return;
  const int b = (int)(index / granules), i = (int)(index % granules);
  int start, count;
  p.pv.rows(b, p.L, start, count);
  if (start < 0) start = 0;
  const int64_t place = (int64_t)(start >> 4) + i;  // granule of the sequence
  const int64_t first = (place << 4) - start;       // row of its first token
  if (first >= p.L) return;
  GatherRows o;
  uint32_t live = 0, zero = 0;
#pragma unroll
  for (int t = 0; t < kGranule; ++t) {
    const int64_t row = first + t;
    if (row >= 0 && row < count) live |= 1u << t;
    if (row >= count && row < p.L && p.zero_padding) zero |= 1u << t;
  }
  const uint8_t *gran = nullptr;
  if (live) {
    gran = granule_of(p.pv, b, (int)min(place << 4, (int64_t)0x7fffffff), kvh, Granule<FMT, D>::kBytes);
    if (!gran) {  // reported; the rows read back as zero
      zero |= live;
      live = 0;
    }
  }
  o.wide = p.wide;
  o.live = live;
  o.zero = zero;
  o.k_sl = p.k_sl;
  o.v_sl = p.v_sl;
  o.k = p.k + b * p.k_sb + first * p.k_sl + kvh * p.k_sh;
  o.v = p.v + b * p.v_sb + first * p.v_sl + kvh * p.v_sh;
  if constexpr (FMT == FPX_PAGES_INT4)
    gather_int4<D>(o, gran, lane);
  else
    gather_bf16<D>(o, gran, lane);
}

// A launch that may begin while the kernel before it ends (each kernel here waits for it).
template <class K, class... A>
static int launch_dependent(K kernel, dim3 grid, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? FPX_OK : FPX_ERR_CUDA;
}

static __device__ int g_bad_index;

// Its address on the current device, looked up once for each.
static int *bad_index_word() {
  static std::atomic<int *> cache[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
  int *word = cache[dev].load(std::memory_order_relaxed);
  if (!word) {
    void *ptr = nullptr;
    if (cudaGetSymbolAddress(&ptr, g_bad_index) != cudaSuccess) return nullptr;
    cache[dev].store(word = static_cast<int *>(ptr), std::memory_order_relaxed);
  }
  return word;
}

int read_bad_index(int *code, int reset) {
  if (cudaMemcpyFromSymbol(code, g_bad_index, sizeof(int)) != cudaSuccess) return FPX_ERR_CUDA;
  const int zero = 0;
  if (reset && cudaMemcpyToSymbol(g_bad_index, &zero, sizeof(int)) != cudaSuccess) return FPX_ERR_CUDA;
  return FPX_OK;
}

int make_page_view(PageView *view, int format, const void *pool, int pages, int page_size, const int32_t *table,
                   int64_t table_stride, int max_pages, const int32_t *starts, const int32_t *counts, int Hkv, int d) {
  if (format != FPX_PAGES_BF16 && format != FPX_PAGES_INT4) return FPX_ERR_INVALID;
  if (!pool || !table || !starts || pages <= 0 || max_pages <= 0 || Hkv <= 0) return FPX_ERR_INVALID;
  if (d != 128 && d != 256) return FPX_ERR_UNSUPPORTED;
  if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1))) return FPX_ERR_UNSUPPORTED;
  if (table_stride < max_pages || (reinterpret_cast<uintptr_t>(pool) & 15)) return FPX_ERR_SHAPE;
  view->pool = static_cast<uint8_t *>(const_cast<void *>(pool));
  view->page_shift = 0;
  while ((16 << view->page_shift) < page_size) ++view->page_shift;
  view->head_bytes = fpx_paged_page_bytes(format, 1, d, page_size);
  view->page_bytes = view->head_bytes * Hkv;
  view->pages = pages;
  view->table = table;
  view->table_stride = table_stride;
  view->max_pages = max_pages;
  view->starts = starts;
  view->counts = counts;
  view->bad_index = bad_index_word();
  return FPX_OK;
}

}  // namespace fpx

using namespace fpx;

extern "C" size_t fpx_paged_page_bytes(int format, int Hkv, int d, int page_size) {
  if (Hkv <= 0 || (d != 128 && d != 256) || page_size < 16 || page_size > 1024 || (page_size & (page_size - 1))) return 0;
  if (format == FPX_PAGES_BF16) return (size_t)Hkv * page_size * 4 * d;
  if (format == FPX_PAGES_INT4) return (size_t)Hkv * page_size * (9 * d / 8 + 2);
  return 0;
}

static bool row_aligned16(const void *p, const RowStrides &s) {
  return !p || (!(reinterpret_cast<uintptr_t>(p) & 15) && s.multiples_of(8));
}
static bool row_aligned(const void *p, const RowStrides &s) {  // 8-byte pieces of a head row
  return !(reinterpret_cast<uintptr_t>(p) & 7) && s.multiples_of(4);
}

extern "C" int fpx_paged_append(int format, const void *q, int64_t q_sb, int64_t q_sl, int64_t q_sh, const void *k,
                                int64_t k_sb, int64_t k_sl, int64_t k_sh, const void *v, int64_t v_sb, int64_t v_sl,
                                int64_t v_sh, int B, int L, int H, int Hkv, int d, const float *rope, int rope_len,
                                int rotary, void *pool, int pages, int page_size, const int32_t *table,
                                int64_t table_stride, int max_pages, const int32_t *starts, const int32_t *counts,
                                void *q_out, int64_t qo_sb, int64_t qo_sl, int64_t qo_sh, void *k_out, int64_t ko_sb,
                                int64_t ko_sl, int64_t ko_sh, int zero_padding, fpx_stream_t stream) {
  FPX_BIND(stream);
  if (!k || !v || B <= 0 || L <= 0 || Hkv <= 0 || H < 0) return FPX_ERR_INVALID;
  if ((H > 0) != (q != nullptr) || (H > 0) != (q_out != nullptr)) return FPX_ERR_INVALID;
  AppendParams p{};
  const int rc = make_page_view(&p.pv, format, pool, pages, page_size, table, table_stride, max_pages, starts, counts,
                               Hkv, d);
  if (rc) return rc;
  if (rope) {
    if (rope_len <= 0) return FPX_ERR_INVALID;
    if (rotary < 8 || rotary > d || rotary % 8 || (reinterpret_cast<uintptr_t>(rope) & 15)) return FPX_ERR_SHAPE;
  }
  const RowStrides qs(q_sb, q_sl, q_sh, B, L, H), ks(k_sb, k_sl, k_sh, B, L, Hkv), vs(v_sb, v_sl, v_sh, B, L, Hkv),
      qo(qo_sb, qo_sl, qo_sh, B, L, H), ko(ko_sb, ko_sl, ko_sh, B, L, Hkv);
  if (!row_aligned(k, ks) || !row_aligned(v, vs) || (H && (!row_aligned(q, qs) || !row_aligned(q_out, qo))) ||
      (k_out && !row_aligned(k_out, ko)))
    return FPX_ERR_SHAPE;
  p.q = static_cast<const __nv_bfloat16 *>(q); p.q_sb = qs.b; p.q_sl = qs.l; p.q_sh = qs.h;
  p.k = static_cast<const __nv_bfloat16 *>(k); p.k_sb = ks.b; p.k_sl = ks.l; p.k_sh = ks.h;
  p.v = static_cast<const __nv_bfloat16 *>(v); p.v_sb = vs.b; p.v_sl = vs.l; p.v_sh = vs.h;
  p.q_out = static_cast<__nv_bfloat16 *>(q_out); p.qo_sb = qo.b; p.qo_sl = qo.l; p.qo_sh = qo.h;
  p.k_out = static_cast<__nv_bfloat16 *>(k_out); p.ko_sb = ko.b; p.ko_sl = ko.l; p.ko_sh = ko.h;
  p.rope = rope; p.rope_len = rope_len; p.rotary = rotary;
  p.B = B; p.L = L; p.H = H; p.Hkv = Hkv; p.zero_padding = zero_padding != 0;
  p.q_wide = row_aligned16(q, qs) && row_aligned16(q_out, qo);
  p.kv_wide = row_aligned16(k, ks) && row_aligned16(v, vs) && row_aligned16(k_out, ko);
  const int64_t blocks = ((int64_t)B * L + 3) / 4;
  // Half the rows a warp where the GPU is not full of warps otherwise (64 tokens: 3.5 -> 2.6 us; 32640: 110 -> 121).
  p.store_rows = (int64_t)B * L * ((2 * Hkv + kStoreRows - 1) / kStoreRows) <= 8 * kSms ? kStoreRows / 2 : kStoreRows;
  const int query_chunks = (H + query_heads(d) - 1) / query_heads(d), chunks = query_chunks + (2 * Hkv + p.store_rows - 1) / p.store_rows;
  if ((int64_t)B * L > 0x7ffffff0 || chunks > 65535) return FPX_ERR_SHAPE;
  const auto kernel = format == FPX_PAGES_INT4
                          ? (d == 256 ? paged_append_kernel<FPX_PAGES_INT4, 256> : paged_append_kernel<FPX_PAGES_INT4, 128>)
                          : (d == 256 ? paged_append_kernel<FPX_PAGES_BF16, 256> : paged_append_kernel<FPX_PAGES_BF16, 128>);
  return launch_dependent(kernel, dim3((unsigned)blocks, chunks), stream, p, query_chunks);
}

extern "C" int fpx_paged_gather(int format, const void *pool, int pages, int page_size, const int32_t *table,
                                int64_t table_stride, int max_pages, const int32_t *starts, const int32_t *counts,
                                int B, int L, int Hkv, int d, void *k, int64_t k_sb, int64_t k_sl, int64_t k_sh,
                                void *v, int64_t v_sb, int64_t v_sl, int64_t v_sh, int zero_padding, fpx_stream_t stream) {
  FPX_BIND(stream);
  if (!k || !v || B <= 0 || L <= 0 || Hkv <= 0) return FPX_ERR_INVALID;
  GatherParams p{};
  const int rc = make_page_view(&p.pv, format, pool, pages, page_size, table, table_stride, max_pages, starts, counts,
                               Hkv, d);
  if (rc) return rc;
  const RowStrides ks(k_sb, k_sl, k_sh, B, L, Hkv), vs(v_sb, v_sl, v_sh, B, L, Hkv);
  if (!row_aligned(k, ks) || !row_aligned(v, vs)) return FPX_ERR_SHAPE;
  p.k = static_cast<__nv_bfloat16 *>(k); p.k_sb = ks.b; p.k_sl = ks.l; p.k_sh = ks.h;
  p.v = static_cast<__nv_bfloat16 *>(v); p.v_sb = vs.b; p.v_sl = vs.l; p.v_sh = vs.h;
  p.B = B; p.L = L; p.Hkv = Hkv; p.zero_padding = zero_padding != 0;
  p.wide = row_aligned16(k, ks) && row_aligned16(v, vs);
  const int granules = L / kGranule + 2;  // that L rows can touch
  const int64_t blocks = ((int64_t)B * granules + 3) / 4;
  if (blocks > 0x7fffffff || Hkv > 65535) return FPX_ERR_SHAPE;
  const auto kernel = format == FPX_PAGES_INT4
                          ? (d == 256 ? paged_gather_kernel<FPX_PAGES_INT4, 256> : paged_gather_kernel<FPX_PAGES_INT4, 128>)
                          : (d == 256 ? paged_gather_kernel<FPX_PAGES_BF16, 256> : paged_gather_kernel<FPX_PAGES_BF16, 128>);
  return launch_dependent(kernel, dim3((unsigned)blocks, Hkv), stream, p, granules);
}
