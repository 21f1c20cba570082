// Writing and reading back the paged KV cache: append (rotary embedding on the way, 4-bit
// quantisation for int4 pages) and gather. Page layout: paged.cuh.
#include <algorithm>

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
  bool zero_padding;
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

FPX_INLINE float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// The four codes of x / s, low nibble first. A scale of zero gives the middle code, 0 * s; so does
// one that is no number or infinite, whose 0 * s is NaN.
FPX_INLINE uint32_t codes4(const float (&x)[4], float s) {
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float n = s > 0.f && s < INFINITY ? fminf(fmaxf(rintf(__fdiv_rn(x[e], s)), -7.f), 7.f) : 0.f;
    w |= (uint32_t)((int)n + 8) << (4 * e);
  }
  return w;
}

// One row of K (VALUE false) or V into the granule of token t.
template <int D, bool VALUE>
FPX_INLINE void write_int4(uint8_t *gran, int t, const float (&x)[D / 128][4], int lane) {
  using G = Granule<FPX_PAGES_INT4, D>;
  const int j = lane >> 3;
  float a[D / 128];
  float top = 0.f;
#pragma unroll
  for (int J = 0; J < D / 128; ++J) {
    float m = max_nan(max_nan(fabsf(x[J][0]), fabsf(x[J][1])), max_nan(fabsf(x[J][2]), fabsf(x[J][3])));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    a[J] = __fdiv_rn(m, 7.f);
    top = max_nan(top, a[J]);
  }
  if (VALUE) {
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 8));
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 16));
    const int e = min(max((int)((__float_as_uint(top) >> 23) & 255u) - 127, -60), 126);
    const float up = __uint_as_float((uint32_t)(e + 127) << 23), down = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
    for (int J = 0; J < D / 128; ++J) {
      const __half r = __float2half_rn(a[J] * down);
      const uint32_t w = codes4(x[J], __half2float(r) * up);
      *reinterpret_cast<uint16_t *>(gran + G::kVCodes + v_chunk(t, J, lane & 7) + 2 * j) = (uint16_t)w;
      if ((lane & 7) == 0)
        *reinterpret_cast<__half *>(gran + G::kVScales + (((t >> 1) * (D / 32) + 4 * J + j) * 2 + (t & 1)) * 2) = r;
    }
    if (lane == 0) *reinterpret_cast<__nv_bfloat16 *>(gran + G::kVExps + 2 * t) = __float2bfloat16_rn((float)e);
  } else {
    const int p = (lane & 7) >> 1;
#pragma unroll
    for (int J = 0; J < D / 128; ++J) {
      const __nv_bfloat16 s = __float2bfloat16_rn(a[J]);
      const uint32_t w = codes4(x[J], __bfloat162float(s));
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

constexpr int kAppendHeads = 4;  // head rows of a warp, loaded before the first is used

// One warp: one token, kAppendHeads consecutive head rows of [q heads | k heads | v heads].
template <int FMT, int D>
__global__ void __launch_bounds__(128) paged_append_kernel(const __grid_constant__ AppendParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t token = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (token >= (int64_t)p.B * p.L) return;
  const int b = (int)(token / p.L), l = (int)(token % p.L);
  const int heads = p.H + 2 * p.Hkv, h0 = blockIdx.y * kAppendHeads;
  const int64_t pos64 = (int64_t)p.pv.starts[b] + l;
  const bool row = l < p.pv.count(b, p.L), past = pos64 > 0x7ffffffe || (p.rope && pos64 >= p.rope_len);
  if (!row || past) {
    if (row) p.pv.fail();
    if (p.zero_padding) {
      const float zero[D / 128][4] = {};
      for (int h = h0; h < min(h0 + kAppendHeads, p.H + p.Hkv); ++h) {
        if (h < p.H)
          store_row<D>(p.q_out + b * p.qo_sb + l * p.qo_sl + h * p.qo_sh, zero, lane);
        else if (p.k_out)
          store_row<D>(p.k_out + b * p.ko_sb + l * p.ko_sl + (h - p.H) * p.ko_sh, zero, lane);
      }
    }
    return;
  }
  const int pos = (int)pos64;
  HeadRow<D> rows[kAppendHeads];
#pragma unroll
  for (int u = 0; u < kAppendHeads; ++u) {
    const int h = h0 + u;
    if (h >= heads) break;
    const __nv_bfloat16 *src = h < p.H ? p.q + b * p.q_sb + l * p.q_sl + h * p.q_sh
                               : h < p.H + p.Hkv ? p.k + b * p.k_sb + l * p.k_sl + (h - p.H) * p.k_sh
                                                 : p.v + b * p.v_sb + l * p.v_sl + (h - p.H - p.Hkv) * p.v_sh;
    rows[u] = load_row<D>(src, lane);
  }
  Turn<D> turn{};
  const int rotary = p.rope ? p.rotary : 0;
  if (p.rope && h0 < p.H + p.Hkv) turn = load_turn<D>(p.rope + (int64_t)pos * rotary, rotary, lane);
  __syncwarp();  // q_out may be q, k_out may be k: a lane stores only after every lane has loaded
#pragma unroll
  for (int u = 0; u < kAppendHeads; ++u) {
    const int h = h0 + u;
    if (h >= heads) break;
    float x[D / 128][4];
    if (h < p.H) {
      rotate_row<D>(rows[u], turn, rotary, lane, x);
      store_row<D>(p.q_out + b * p.qo_sb + l * p.qo_sl + h * p.qo_sh, x, lane);
      continue;
    }
    const bool value = h >= p.H + p.Hkv;
    const int kvh = h - p.H - (value ? p.Hkv : 0);
    if (value)
      unpack_row<D>(rows[u], x);
    else
      rotate_row<D>(rows[u], turn, rotary, lane, x);
    if (!value && p.k_out) store_row<D>(p.k_out + b * p.ko_sb + l * p.ko_sl + kvh * p.ko_sh, x, lane);
    uint8_t *gran = granule_of(p.pv, b, pos, kvh, Granule<FMT, D>::kBytes);
    if (!gran) continue;
    const int t = pos & (kGranule - 1);
    if (FMT == FPX_PAGES_INT4) {
      if (value)
        write_int4<D, true>(gran, t, x, lane);
      else
        write_int4<D, false>(gran, t, x, lane);
    } else {
      if (value)
        write_bf16<D, true>(gran, t, x, lane);
      else
        write_bf16<D, false>(gran, t, x, lane);
    }
  }
}

struct GatherParams {
  PageView pv;
  __nv_bfloat16 *k, *v;
  int64_t k_sb, k_sl, k_sh, v_sb, v_sl, v_sh;
  int B, L, Hkv;
  bool zero_padding;
};

// One warp: one token and KV head.
template <int FMT, int D>
__global__ void __launch_bounds__(128) paged_gather_kernel(const __grid_constant__ GatherParams p) {
  using G = Granule<FMT, D>;
  const int lane = threadIdx.x & 31, kvh = blockIdx.y;
  const int64_t token = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (token >= (int64_t)p.B * p.L) return;
  const int b = (int)(token / p.L), l = (int)(token % p.L);
  const bool row = l < p.pv.count(b, p.L);
  if (!row && !p.zero_padding) return;
  const int pos = (int)min((int64_t)p.pv.starts[b] + l, (int64_t)0x7fffffff), t = pos & (kGranule - 1);
  const uint8_t *gran = row ? granule_of(p.pv, b, pos, kvh, G::kBytes) : nullptr;
  __nv_bfloat16 *ko = p.k + b * p.k_sb + l * p.k_sl + kvh * p.k_sh, *vo = p.v + b * p.v_sb + l * p.v_sl + kvh * p.v_sh;
  float k[D / 128][4] = {}, v[D / 128][4] = {};
  if (gran) {
    if constexpr (FMT == FPX_PAGES_BF16) {
      HeadRow<D> kr, vr;
#pragma unroll
      for (int J = 0; J < D / 128; ++J) {
        const int at = t * G::kRow + (((16 * J + (lane >> 1)) ^ (t & 7)) << 4) + ((lane & 1) << 3);
        kr.w[J] = *reinterpret_cast<const uint2 *>(gran + at);
        vr.w[J] = *reinterpret_cast<const uint2 *>(gran + at + 2 * D);
      }
      unpack_row<D>(kr, k);
      unpack_row<D>(vr, v);
    } else {
      const int j = lane >> 3, part = (lane & 7) >> 1;
      const float e = __bfloat162float(*reinterpret_cast<const __nv_bfloat16 *>(gran + G::kVExps + 2 * t));
      const float up = __uint_as_float((uint32_t)((int)e + 127) << 23);
#pragma unroll
      for (int J = 0; J < D / 128; ++J) {
        const uint32_t kc = *reinterpret_cast<const uint16_t *>(gran + t * (D / 2) + J * 64 + (4 * part + j) * 4 + (lane & 1) * 2);
        const uint32_t vc = *reinterpret_cast<const uint16_t *>(gran + G::kVCodes + v_chunk(t, J, lane & 7) + 2 * j);
        const float ks = __bfloat162float(*reinterpret_cast<const __nv_bfloat16 *>(gran + G::kKScales + (t * (D / 32) + 4 * J + j) * 2));
        const float vs = __half2float(*reinterpret_cast<const __half *>(gran + G::kVScales + (((t >> 1) * (D / 32) + 4 * J + j) * 2 + (t & 1)) * 2)) * up;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          k[J][i] = (float)((int)((kc >> (4 * i)) & 15u) - 8) * ks;
          v[J][i] = (float)((int)((vc >> (4 * i)) & 15u) - 8) * vs;
        }
      }
    }
  }
  store_row<D>(ko, k, lane);
  store_row<D>(vo, v, lane);
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
  view->error = device_error_word();
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
  const int64_t blocks = ((int64_t)B * L + 3) / 4;
  const int chunks = (H + 2 * Hkv + kAppendHeads - 1) / kAppendHeads;
  if (blocks > 0x7fffffff || chunks > 65535) return FPX_ERR_SHAPE;
  const dim3 grid((unsigned)blocks, chunks);
  if (format == FPX_PAGES_INT4) {
    if (d == 256)
      paged_append_kernel<FPX_PAGES_INT4, 256><<<grid, 128, 0, stream>>>(p);
    else
      paged_append_kernel<FPX_PAGES_INT4, 128><<<grid, 128, 0, stream>>>(p);
  } else {
    if (d == 256)
      paged_append_kernel<FPX_PAGES_BF16, 256><<<grid, 128, 0, stream>>>(p);
    else
      paged_append_kernel<FPX_PAGES_BF16, 128><<<grid, 128, 0, stream>>>(p);
  }
  FPX_CHECK_LAUNCH();
  return FPX_OK;
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
  const int64_t blocks = ((int64_t)B * L + 3) / 4;
  if (blocks > 0x7fffffff || Hkv > 65535) return FPX_ERR_SHAPE;
  const dim3 grid((unsigned)blocks, Hkv);
  if (format == FPX_PAGES_INT4) {
    if (d == 256)
      paged_gather_kernel<FPX_PAGES_INT4, 256><<<grid, 128, 0, stream>>>(p);
    else
      paged_gather_kernel<FPX_PAGES_INT4, 128><<<grid, 128, 0, stream>>>(p);
  } else {
    if (d == 256)
      paged_gather_kernel<FPX_PAGES_BF16, 256><<<grid, 128, 0, stream>>>(p);
    else
      paged_gather_kernel<FPX_PAGES_BF16, 128><<<grid, 128, 0, stream>>>(p);
  }
  FPX_CHECK_LAUNCH();
  return FPX_OK;
}
