// Decode attention over the paged KV cache (bf16 or 4-bit pages), causal by position: row i of
// sequence b stands at starts[b] + i and sees the cached tokens up to and with itself.
//
// out[row] = sum_t p_t v_t / sum_t p_t, p_t = exp2(s_t - m), s_t = (q . k_t) scale log2 e.
//
// The pages are read once, so HBM bounds the long cases; the rest of the design keeps the
// 4-bit arithmetic below that. The G query heads of a KV head (x rows of the call) are the
// *columns* of both products, S^T = K Q^T and O^T = V^T P^T: keys are the 16 rows of
// mma.sync's A operand, which 4-bit codes expand into straight from shared memory in the
// layout paged.cuh describes, and 8 columns waste little for the usual groups of 4 to 8.
//   K: code n becomes the bf16 128 + n by one and-or (0x4300 | n); the offset 136 = 128 + 8 is
//      taken out in the accumulator's start value, -136 sum(q) over the group, and the group's
//      scale multiplies the group's sum.
//   V: codes become the fp16 n - 8 (two logic operations and one exact fma a pair); the scales
//      r < 2 multiply the probabilities, in fp16 (11 bits: its rounding stays below the bf16 of the
//      output). The row exponent 2^e joins the logit: u = exp2(s + e - m) <= 2^8 whatever the
//      values' size, and the sum of weights takes u 2^-e.
//   bf16 pages: P is split in two bf16 terms, so that it does not round before the output does.
//
// Work is split evenly over the CTAs of one launch, whatever the sequences' lengths: the
// steps (one or two granules of 16 tokens) of all (sequence, row block, KV head) units lie end to
// end, each CTA takes an equal run of them, and its four warps every fourth step, each through its own
// ring of bulk copies (no barrier between warps inside a unit). A unit inside one CTA is
// finished there; the pieces of the others are merged in CTA order by the second launch, so
// results do not depend on timing.
#include <algorithm>

#include "paged.cuh"
#include "tc.cuh"

namespace fpx {

struct PagedDecodeParams {
  PageView pv;
  const __nv_bfloat16 *q;
  int64_t q_sb, q_sl, q_sh;
  __nv_bfloat16 *out;
  int64_t o_sb, o_sl, o_sh;
  float *lse;  // [B][Lq][H] or null
  int B, Lq, H, Hkv, group, blocks;  // blocks: row blocks of 8 NT (query row, head of the group) pairs
  float scale_log2;
  int ctas, min_steps;
  int *prefix;     // [B * blocks + 1] steps of all heads before an item (b, row block)
  float *part_o;   // [ctas + units][8 NT][d]
  float *part_ml;  // [ctas + units][8 NT][2]
};

constexpr float kRaise = 8.f;      // the running reference follows when a logit passes it by this (log2)
constexpr float kLowest = -3e38f;  // reference before any logit: below all of them, and finite

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
FPX_INLINE int steps_of(int keys) { return (keys + GS * kGranule - 1) / (GS * kGranule); }

FPX_INLINE uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
FPX_INLINE uint32_t transpose8(uint32_t a) {  // 8 x 8 16-bit matrix, one row of pairs a quad
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
FPX_INLINE void mma_f16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
FPX_INLINE void mma_bf16_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {  // D = A B
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
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
FPX_INLINE uint4 lds128(const uint8_t *p) { return *reinterpret_cast<const uint4 *>(p); }
FPX_INLINE void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

template <int FMT, int D, int NT, int GS, int W, int ST>
struct PagedSmem {
  union {
    uint8_t ring[W][ST][GS * Granule<FMT, D>::kBytes];
    struct {
      float o[W][8 * NT][D];
      float m[W][8 * NT], l[W][8 * NT];
    } merge;
  };
  uint64_t full[W][ST];
  int scan[W];
  int item, base, abort;
};

// The warp's share of a unit: its columns' running reference m, sums l and O^T.
template <int D, int NT>
struct Columns {
  float o[D / 16][NT][4];
  float m[NT][2], l[NT][2];
};

// Raises the reference m where a logit has passed it by kRaise (always on a first finite logit),
// and rescales what was summed under the old one.
template <int D, int NT, int GS>
FPX_INLINE void follow(Columns<D, NT> &c, const float (&y)[GS][NT][4]) {
  float top[NT][2];
  bool up = false;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      top[n][e] = fmaxf(y[0][n][e], y[0][n][e + 2]);
#pragma unroll
      for (int h = 1; h < GS; ++h) top[n][e] = tc::fmax3(top[n][e], y[h][n][e], y[h][n][e + 2]);
      up |= top[n][e] > c.m[n][e] + kRaise;
    }
  if (!__any_sync(0xffffffffu, up)) return;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float x = top[n][e];
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
      const float m = fmaxf(c.m[n][e], x);
      const float keep = tc::ex2(c.m[n][e] - m);
      c.m[n][e] = m;
      c.l[n][e] *= keep;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        c.o[i][n][e] *= keep;
        c.o[i][n][e + 2] *= keep;
      }
    }
}

// Query fragments of a unit (B operands of S^T = K Q^T), column n = lane / 4 of each tile.
template <int FMT, int D, int NT>
struct Queries {
  uint32_t b[D / 16][NT][2];
  // int4: the codes' offset, -136 sum(q) of each group, as three bf16 terms: it multiplies the groups' scales in one more
  // product of four groups x (high, middle, low) for every 128 dims
  uint32_t off[FMT == FPX_PAGES_INT4 ? D / 128 : 1][NT][2];
};
template <int FMT, int D, int NT>
FPX_INLINE void load_queries(Queries<FMT, D, NT> &f, const PagedDecodeParams &p, int b, int row0, int rows, int kvh,
                             int lane) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = row0 + 8 * n + g;
    const bool live = r < rows;
    const __nv_bfloat16 *q = p.q + b * p.q_sb + (int64_t)(live ? r / p.group : 0) * p.q_sl +
                             (int64_t)(kvh * p.group + (live ? r % p.group : 0)) * p.q_sh;
    if constexpr (FMT == FPX_PAGES_INT4) {
      uint4 w[D / 32];
#pragma unroll
      for (int j = 0; j < D / 32; ++j)
        w[j] = live ? *reinterpret_cast<const uint4 *>(q + 32 * j + 8 * t) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int J = 0; J < D / 128; ++J) {
        float sum[4];
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
          const int j = 4 * J + jj;
          // the codes' pairs are (i, i + 4) of a lane's eight dims
          f.b[2 * j][n][0] = __byte_perm(w[j].x, w[j].z, 0x5410);
          f.b[2 * j][n][1] = __byte_perm(w[j].x, w[j].z, 0x7632);
          f.b[2 * j + 1][n][0] = __byte_perm(w[j].y, w[j].w, 0x5410);
          f.b[2 * j + 1][n][1] = __byte_perm(w[j].y, w[j].w, 0x7632);
          const uint32_t v[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
          float x = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) x += __uint_as_float(v[i] << 16) + __uint_as_float(v[i] & 0xffff0000u);
          x += __shfl_xor_sync(0xffffffffu, x, 1);
          x += __shfl_xor_sync(0xffffffffu, x, 2);
          sum[jj] = -136.f * x;
        }
        // k = 2 t, 2 t + 1 of the product: groups 2 (t & 1), + 1; terms high (t < 2), middle; k + 8: low, none
        const float x0 = t & 1 ? sum[2] : sum[0], x1 = t & 1 ? sum[3] : sum[1];
        const float h0 = __bfloat162float(__float2bfloat16_rn(x0)), h1 = __bfloat162float(__float2bfloat16_rn(x1));
        const float m0 = __bfloat162float(__float2bfloat16_rn(x0 - h0)), m1 = __bfloat162float(__float2bfloat16_rn(x1 - h1));
        f.off[J][n][0] = t < 2 ? pack_bf16(h0, h1) : pack_bf16(m0, m1);
        f.off[J][n][1] = t < 2 ? pack_bf16(x0 - h0 - m0, x1 - h1 - m1) : 0u;
      }
    } else {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        f.b[kk][n][0] = live ? *reinterpret_cast<const uint32_t *>(q + 16 * kk + 2 * t) : 0u;
        f.b[kk][n][1] = live ? *reinterpret_cast<const uint32_t *>(q + 16 * kk + 8 + 2 * t) : 0u;
      }
    }
  }
}

// S^T of one granule: y[n] = keys (g, g + 8) x columns (2 t, 2 t + 1), without the softmax's scale.
template <int FMT, int D, int NT>
FPX_INLINE void scores(float (&y)[NT][4], const Queries<FMT, D, NT> &f, const uint8_t *gran, int lane) {
  using G = Granule<FMT, D>;
  const int g = lane >> 2, t = lane & 3;
  if constexpr (FMT == FPX_PAGES_INT4) {
#pragma unroll
    for (int J = 0; J < D / 128; ++J) {
      const uint4 ka = lds128(gran + g * (D / 2) + J * 64 + t * 16), kb = lds128(gran + (g + 8) * (D / 2) + J * 64 + t * 16);
      const uint2 sa = *reinterpret_cast<const uint2 *>(gran + G::kKScales + g * (D / 16) + 8 * J);
      const uint2 sb = *reinterpret_cast<const uint2 *>(gran + G::kKScales + (g + 8) * (D / 16) + 8 * J);
      const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
      {
        const uint32_t xa = t & 1 ? sa.y : sa.x, xb = t & 1 ? sb.y : sb.x;
        const uint32_t a[4] = {xa, xb, xa, xb};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (J == 0)
            mma_bf16_zero(y[n], a, f.off[J][n][0], f.off[J][n][1]);
          else
            mma_bf16_16816(y[n], a, f.off[J][n][0], f.off[J][n][1]);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t lo = 0x000f000fu, one = 0x43004300u;  // bf16 128 + n
        const uint32_t a0[4] = {and_or(wa[j], lo, one), and_or(wb[j], lo, one), and_or(wa[j] >> 4, lo, one),
                                and_or(wb[j] >> 4, lo, one)};
        const uint32_t a1[4] = {and_or(wa[j] >> 8, lo, one), and_or(wb[j] >> 8, lo, one), and_or(wa[j] >> 12, lo, one),
                                and_or(wb[j] >> 12, lo, one)};
        const uint32_t ua = j < 2 ? sa.x : sa.y, ub = j < 2 ? sb.x : sb.y;
        const float fa = __uint_as_float(j & 1 ? ua & 0xffff0000u : ua << 16);
        const float fb = __uint_as_float(j & 1 ? ub & 0xffff0000u : ub << 16);
        const int gr = 4 * J + j;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float acc[4];
          mma_bf16_zero(acc, a0, f.b[2 * gr][n][0], f.b[2 * gr][n][1]);
          mma_bf16_16816(acc, a1, f.b[2 * gr + 1][n][0], f.b[2 * gr + 1][n][1]);
          y[n][0] = fmaf(fa, acc[0], y[n][0]);
          y[n][1] = fmaf(fa, acc[1], y[n][1]);
          y[n][2] = fmaf(fb, acc[2], y[n][2]);
          y[n][3] = fmaf(fb, acc[3], y[n][3]);
        }
      }
    }
  } else {
    const int r = (lane & 7) + (lane & 8), hi = lane >> 4;
#pragma unroll
    for (int n = 0; n < NT; ++n) y[n][0] = y[n][1] = y[n][2] = y[n][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      uint32_t a[4];
      ldmatrix_x4(a[0], a[1], a[2], a[3], smem_u32(gran + r * G::kRow + (((2 * kk + hi) ^ (r & 7)) << 4)));
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_bf16_16816(y[n], a, f.b[kk][n][0], f.b[kk][n][1]);
    }
  }
}

// O^T += V^T P^T of one granule; y: the probabilities; wa, wb: 2^-e of the two keys (int4). EDGE: tokens
// from `have` on are not there (unseen, or on a missing page), and may hold anything.
template <int FMT, int D, int NT, bool EDGE>
FPX_INLINE void values(Columns<D, NT> &c, const float (&y)[NT][4], float wa, float wb, uint8_t *gran, int have, int lane) {
  using G = Granule<FMT, D>;
  const int g = lane >> 2, t = lane & 3;
  if constexpr (FMT == FPX_PAGES_INT4) {
    uint32_t pb[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      c.l[n][0] = fmaf(y[n][0], wa, fmaf(y[n][2], wb, c.l[n][0]));
      c.l[n][1] = fmaf(y[n][1], wa, fmaf(y[n][3], wb, c.l[n][1]));
      pb[n][0] = transpose8(pack_f16(y[n][0], y[n][1]));
      pb[n][1] = transpose8(pack_f16(y[n][2], y[n][3]));
    }
    const uint32_t keep0 = (2 * t < have ? 0xffffu : 0u) | (2 * t + 1 < have ? 0xffff0000u : 0u);
    const uint32_t keep1 = (2 * t + 8 < have ? 0xffffu : 0u) | (2 * t + 9 < have ? 0xffff0000u : 0u);
#pragma unroll
    for (int J = 0; J < D / 128; ++J) {
      const uint4 va = lds128(gran + G::kVCodes + v_chunk(2 * t, J, g)), vb = lds128(gran + G::kVCodes + v_chunk(2 * t + 8, J, g));
      const uint4 ra = lds128(gran + G::kVScales + t * (D / 8) + 16 * J), rb = lds128(gran + G::kVScales + (t + 4) * (D / 8) + 16 * J);
      const uint32_t r0[4] = {ra.x, ra.y, ra.z, ra.w}, r1[4] = {rb.x, rb.y, rb.z, rb.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t sel = j & 1 ? 0x7632 : 0x5410;  // the same four dims of the even and of the odd token
        const uint32_t u0 = j < 2 ? __byte_perm(va.x, va.z, sel) : __byte_perm(va.y, va.w, sel);
        const uint32_t u1 = j < 2 ? __byte_perm(vb.x, vb.z, sel) : __byte_perm(vb.y, vb.w, sel);
        const uint32_t lo = 0x000f000fu, hi = 0x00f000f0u, k = 0x64006400u;  // fp16 1024 + n, 1024 + 16 n
        const uint32_t off = 0x64086408u, sixteenth = 0x2c002c00u, m72 = 0xd480d480u;  // 1032, 1 / 16, -72
        const uint32_t a0[4] = {hsub2u(and_or(u0, lo, k), off), hfma2u(and_or(u0, hi, k), sixteenth, m72),
                                hsub2u(and_or(u1, lo, k), off), hfma2u(and_or(u1, hi, k), sixteenth, m72)};
        const uint32_t a1[4] = {hsub2u(and_or(u0 >> 8, lo, k), off), hfma2u(and_or(u0 >> 8, hi, k), sixteenth, m72),
                                hsub2u(and_or(u1 >> 8, lo, k), off), hfma2u(and_or(u1 >> 8, hi, k), sixteenth, m72)};
        const int i = 8 * J + 2 * j;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint32_t b0 = hmul2u(pb[n][0], EDGE ? r0[j] & keep0 : r0[j]), b1 = hmul2u(pb[n][1], EDGE ? r1[j] & keep1 : r1[j]);
          mma_f16_16816(c.o[i][n], a0, b0, b1);
          mma_f16_16816(c.o[i + 1][n], a1, b0, b1);
        }
      }
    }
  } else {
    uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float x0 = y[n][2 * e], x1 = y[n][2 * e + 1];
        c.l[n][0] += x0;
        c.l[n][1] += x1;
        const uint32_t h = pack_bf16(x0, x1);
        ph[n][e] = transpose8(h);
        pl[n][e] = transpose8(pack_bf16(x0 - __uint_as_float(h << 16), x1 - __uint_as_float(h & 0xffff0000u)));
      }
    const int r = (lane & 7) + ((lane >> 4) << 3), hi = (lane >> 3) & 1;
    if (EDGE) {
      for (int i = lane; i < kGranule * (D / 8); i += 32) {
        const int row = i / (D / 8);
        if (row >= have) *reinterpret_cast<uint4 *>(gran + row * G::kRow + 2 * D + 16 * (i % (D / 8))) = make_uint4(0, 0, 0, 0);
      }
      __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      uint32_t a[4];
      ldmatrix_x4_trans(a[0], a[1], a[2], a[3], smem_u32(gran + r * G::kRow + 2 * D + (((2 * i + hi) ^ (r & 7)) << 4)));
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mma_bf16_16816(c.o[i][n], a, ph[n][0], ph[n][1]);
        mma_bf16_16816(c.o[i][n], a, pl[n][0], pl[n][1]);
      }
    }
  }
}

// One step: GS granules from key0 on. EDGE: the unit's rows see only keys below `seen`, this lane's
// columns those below limit, and the granules of `dead` are on missing pages.
template <int FMT, int D, int NT, int GS, bool EDGE>
FPX_INLINE void attend_step(Columns<D, NT> &c, const Queries<FMT, D, NT> &f, uint8_t *stage, int key0, int seen,
                            const int (&limit)[NT][2], uint32_t dead, float scale_log2, int lane) {
  using G = Granule<FMT, D>;
  const int g = lane >> 2;
  float y[GS][NT][4], w[GS][2];
  int have[GS];
#pragma unroll
  for (int h = 0; h < GS; ++h) {
    uint8_t *gran = stage + h * G::kBytes;
    scores<FMT, D, NT>(y[h], f, gran, lane);
    have[h] = !EDGE ? kGranule : (dead >> h) & 1 ? 0 : max(0, seen - key0 - kGranule * h);
    w[h][0] = w[h][1] = 1.f;
    float e[2] = {0.f, 0.f};  // row exponents of the two keys' values
    if constexpr (FMT == FPX_PAGES_INT4) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        e[i] = __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t *>(gran + G::kVExps + 2 * g + 16 * i) << 16);
        if (EDGE && g + 8 * i >= have[h]) e[i] = 0.f;
        w[h][i] = tc::ex2(-e[i]);
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y[h][n][i] = fmaf(y[h][n][i], scale_log2, e[i >> 1]);
        const int k = g + 8 * (i >> 1);
        if (EDGE && (k >= have[h] || key0 + kGranule * h + k >= limit[n][i & 1])) y[h][n][i] = -INFINITY;
      }
  }
  follow<D, NT, GS>(c, y);
#pragma unroll
  for (int h = 0; h < GS; ++h) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) y[h][n][i] = tc::ex2(y[h][n][i] - c.m[n][i & 1]);
    values<FMT, D, NT, EDGE>(c, y[h], w[h][0], w[h][1], stage + h * G::kBytes, have[h], lane);
  }
}

// Dim of O^T row `row` (0 or 8 + g: the accumulator's two rows) of tile i: the V codes' layout
// gives a lane four neighbouring dims over two tiles, ldmatrix the plain order.
template <int FMT>
FPX_INLINE int out_dim(int i, int g, int second) {
  return FMT == FPX_PAGES_INT4 ? 16 * (i & ~1) + 4 * g + 2 * (i & 1) + second : 16 * i + 8 * second + g;
}

template <int FMT, int D, int NT, int GS, int W, int ST, int OCC>
__global__ void __launch_bounds__(32 * W, OCC) paged_decode_kernel(const __grid_constant__ PagedDecodeParams p) {
  using G = Granule<FMT, D>;
  using Smem = PagedSmem<FMT, D, NT, GS, W, ST>;
  constexpr int kStep = GS * kGranule, kBytes = GS * G::kBytes;
  constexpr uint32_t kAll = (1u << GS) - 1;
  constexpr int kRows = 8 * NT, kThreads = 32 * W;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Smem &sh = *reinterpret_cast<Smem *>(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int items = p.B * p.blocks;
  if (lane < ST) tc::mbar_init(&sh.full[warp][lane], 1);
  if (tid == 0) sh.abort = 0;
  tc::fence_barrier_init();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // This CTA's run of steps, and the item that it starts in.
  const int chunk = (items + kThreads - 1) / kThreads;
  const int i0 = min(items, tid * chunk), i1 = min(items, i0 + chunk);
  auto steps_in = [&](int i) {
    const int b = i / p.blocks;
    int start, count;
    p.pv.rows(b, p.Lq, start, count);
    return steps_of<GS>(item_keys<NT>(p, start, count, i - b * p.blocks)) * p.Hkv;
  };
  int mine = 0;
  for (int i = i0; i < i1; ++i) mine += steps_in(i);
  int before = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += x;
  }
  if (lane == 31) sh.scan[warp] = before;
  before -= mine;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w < warp) before += sh.scan[w];
    total += sh.scan[w];
  }
  if (blockIdx.x == 0) {  // for the merge
    int at = before;
    for (int i = i0; i < i1; ++i) {
      p.prefix[i] = at;
      at += chunk == 1 ? mine : steps_in(i);
    }
    if (tid == 0) p.prefix[items] = total;
  }
  const int per = max(p.min_steps, (total + p.ctas - 1) / p.ctas);
  int lo = (int)min((int64_t)blockIdx.x * per, (int64_t)total);
  const int hi = min(total, lo + per);
  if (lo >= hi) return;
  if (before <= lo && lo < before + mine) {
    int at = before;
    for (int i = i0; i < i1; ++i) {
      const int n = chunk == 1 ? mine : steps_in(i);
      if (lo < at + n) {
        sh.item = i;
        sh.base = at;
        break;
      }
      at += n;
    }
  }
  __syncthreads();

  int item = sh.item, base = sh.base;
  uint32_t issued = 0, taken = 0, dead = 0;  // steps through this warp's ring; dead: GS bits a stage
  bool stopped = false;
  while (lo < hi) {
    const int b = item / p.blocks, rb = item - b * p.blocks;
    int start, count;
    p.pv.rows(b, p.Lq, start, count);
    const int seen = item_keys<NT>(p, start, count, rb), n_steps = steps_of<GS>(seen);
    if (lo - base >= n_steps * p.Hkv) {  // hi > lo: another item has steps left
      base += n_steps * p.Hkv;
      ++item;
      continue;
    }
    const int kvh = (lo - base) / n_steps, g0 = (lo - base) - kvh * n_steps;
    const int g1 = min(n_steps, g0 + (hi - lo));
    const int rows = count * p.group, row0 = rb * kRows;

    // Ring: copy step g0 + warp + W i into stage (issued mod ST).
    const int32_t *table = p.pv.table + (int64_t)b * p.pv.table_stride;
    const uint8_t *heads = p.pv.pool + (int64_t)kvh * p.pv.head_bytes;
    const int todo = g1 - g0 > warp ? (g1 - g0 - warp + W - 1) / W : 0;
    const int last_page = (seen - 1) >> (p.pv.page_shift + 4);
    int sent = 0, page = 0;
    auto issue = [&]() {
      const int first = GS * (g0 + warp + W * sent);  // granule
      const int st = issued % ST;
      uint64_t *bar = &sh.full[warp][st];
      uint8_t *dst = sh.ring[warp][st];
      if (GS == 1 || p.pv.page_shift > 0) {  // all granules on one page
        if ((sent & 31) == 0) page = table[min((GS * (g0 + warp + W * (sent + lane))) >> p.pv.page_shift, last_page)];
        const int pg = __shfl_sync(0xffffffffu, page, sent & 31);
        const bool ok = (unsigned)pg < (unsigned)p.pv.pages;
        dead = (dead & ~(kAll << (GS * st))) | (ok ? 0u : kAll << (GS * st));
        if (lane == 0) {
          if (!ok) p.pv.fail();
          tc::mbar_expect_tx(bar, kBytes);
          bulk_load(dst, heads + (int64_t)(ok ? pg : 0) * p.pv.page_bytes + (first & ((1 << p.pv.page_shift) - 1)) * G::kBytes,
                    kBytes, bar);
        }
      } else {  // a page each; the second granule of a sequence's last step may not exist
        if ((sent & 15) == 0) page = table[min(2 * (g0 + warp + W * (sent + (lane >> 1))) + (lane & 1), last_page)];
        const bool both = first + 1 <= last_page;
        const int pa = __shfl_sync(0xffffffffu, page, 2 * (sent & 15)), pb = __shfl_sync(0xffffffffu, page, 2 * (sent & 15) + 1);
        const bool oka = (unsigned)pa < (unsigned)p.pv.pages, okb = both && (unsigned)pb < (unsigned)p.pv.pages;
        dead = (dead & ~(kAll << (GS * st))) | ((oka ? 0u : 1u) | (okb ? 0u : 2u)) << (GS * st);
        if (lane == 0) {
          if (!oka || (both && !okb)) p.pv.fail();
          tc::mbar_expect_tx(bar, (okb ? 2 : 1) * G::kBytes);
          bulk_load(dst, heads + (int64_t)(oka ? pa : 0) * p.pv.page_bytes, G::kBytes, bar);
          if (okb) bulk_load(dst + G::kBytes, heads + (int64_t)pb * p.pv.page_bytes, G::kBytes, bar);
        }
      }
      ++issued;
      ++sent;
    };
    while (sent < min(todo, ST) && !stopped) issue();

    Queries<FMT, D, NT> f;
    load_queries<FMT, D, NT>(f, p, b, row0, rows, kvh, lane);
    int limit[NT][2], least = seen;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = row0 + 8 * n + 2 * t + e;
        limit[n][e] = r < rows ? (int)min((int64_t)seen, (int64_t)start + r / p.group + 1) : seen;
        least = min(least, limit[n][e]);
      }
    least = min(least, __shfl_xor_sync(0xffffffffu, least, 1));
    least = min(least, __shfl_xor_sync(0xffffffffu, least, 2));
    Columns<D, NT> c;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      c.m[n][0] = c.m[n][1] = kLowest;
      c.l[n][0] = c.l[n][1] = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) c.o[i][n][0] = c.o[i][n][1] = c.o[i][n][2] = c.o[i][n][3] = 0.f;
    }
    for (int i = 0; i < todo && !stopped; ++i) {
      const int st = taken % ST;
      if (!tc::mbar_wait_warp(&sh.full[warp][st], (taken / ST) & 1, &sh.abort)) {
        stopped = true;  // the copy did not arrive: report it and let the launch end
        if (lane == 0 && p.pv.error) atomicMax(p.pv.error, FPX_DEVICE_WAIT);
        break;
      }
      ++taken;
      const int key0 = (g0 + warp + W * i) * kStep;
      const uint32_t gone = (dead >> (GS * st)) & kAll;
      if (key0 + kStep <= least && !gone)
        attend_step<FMT, D, NT, GS, false>(c, f, sh.ring[warp][st], key0, seen, limit, 0u, p.scale_log2, lane);
      else
        attend_step<FMT, D, NT, GS, true>(c, f, sh.ring[warp][st], key0, seen, limit, gone, p.scale_log2, lane);
      if (sent < todo) {
        // the step's reads (and the zeros written over unseen values) come before the next copy into the stage
        if (FMT == FPX_PAGES_BF16) tc::fence_proxy_async();
        __syncwarp();
        issue();
      }
    }
    if (stopped)  // copies still in flight end before this memory is used again, or this long later
      for (; taken < issued; ++taken) {
        const long long from = clock64();
        while (!tc::mbar_test(&sh.full[warp][taken % ST], (taken / ST) & 1) && clock64() - from < tc::kWaitCycles) {
        }
      }

    // Merge the warps through the ring's memory.
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        c.l[n][e] += __shfl_xor_sync(0xffffffffu, c.l[n][e], 4);
        c.l[n][e] += __shfl_xor_sync(0xffffffffu, c.l[n][e], 8);
        c.l[n][e] += __shfl_xor_sync(0xffffffffu, c.l[n][e], 16);
      }
    __syncthreads();  // every warp has read its last step
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = 8 * n + 2 * t + e;
        if (g == 0) {
          sh.merge.m[warp][col] = c.m[n][e];
          sh.merge.l[warp][col] = c.l[n][e];
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          sh.merge.o[warp][col][out_dim<FMT>(i, g, 0)] = c.o[i][n][e];
          sh.merge.o[warp][col][out_dim<FMT>(i, g, 1)] = c.o[i][n][e + 2];
        }
      }
    __syncthreads();
    const bool whole = g0 == 0 && g1 == n_steps;
    const int64_t slot = blockIdx.x + (int64_t)item * p.Hkv + kvh;
    constexpr int kQuads = D / 4;
    for (int i = tid; i < kRows * kQuads; i += kThreads) {
      const int r = i / kQuads, d = 4 * (i % kQuads);
      if (row0 + r >= rows) break;
      float m = sh.merge.m[0][r], l = 0.f;
#pragma unroll
      for (int w = 1; w < W; ++w) m = fmaxf(m, sh.merge.m[w][r]);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float s = tc::ex2(sh.merge.m[w][r] - m);
        const float4 x = *reinterpret_cast<const float4 *>(&sh.merge.o[w][r][d]);
        l = fmaf(sh.merge.l[w][r], s, l);
        o.x = fmaf(x.x, s, o.x); o.y = fmaf(x.y, s, o.y); o.z = fmaf(x.z, s, o.z); o.w = fmaf(x.w, s, o.w);
      }
      if (whole) {
        const int row = (row0 + r) / p.group, h = kvh * p.group + (row0 + r) % p.group;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        __nv_bfloat16 *out = p.out + b * p.o_sb + row * p.o_sl + h * p.o_sh + d;
        out[0] = __float2bfloat16_rn(o.x * inv); out[1] = __float2bfloat16_rn(o.y * inv);
        out[2] = __float2bfloat16_rn(o.z * inv); out[3] = __float2bfloat16_rn(o.w * inv);
        if (p.lse && d == 0) p.lse[((int64_t)b * p.Lq + row) * p.H + h] = l == 0.f ? -INFINITY : m * kLn2 + logf(l);
      } else {
        *reinterpret_cast<float4 *>(&p.part_o[(slot * kRows + r) * D + d]) = o;
        if (d == 0) *reinterpret_cast<float2 *>(&p.part_ml[2 * (slot * kRows + r)]) = make_float2(m, l);
      }
    }
    tc::fence_proxy_async();  // these accesses of shared memory come before the next unit's copies
    __syncthreads();
    lo += g1 - g0;
  }
}

// Merges the pieces of one (unit, row): D / 4 threads a piece, kPieces of them at a time. Rows
// that see nothing (padding, inactive sequences) become zero here.
constexpr int kMergeThreads = 256;
template <int D, int NT>
__global__ void __launch_bounds__(kMergeThreads) paged_merge_kernel(const __grid_constant__ PagedDecodeParams p) {
  constexpr int kPieces = kMergeThreads / (D / 4), kRows = 8 * NT;
  const int r = blockIdx.y, kvh = blockIdx.x % p.Hkv, item = blockIdx.x / p.Hkv;
  const int b = item / p.blocks, rr = (item % p.blocks) * kRows + r;
  const int row = rr / p.group, h = kvh * p.group + rr % p.group;
  const int tid = threadIdx.x, piece = tid / (D / 4), d = 4 * (tid % (D / 4));
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (rr >= p.Lq * p.group) return;
  int start, count;
  p.pv.rows(b, p.Lq, start, count);
  __nv_bfloat16 *out = p.out + b * p.o_sb + row * p.o_sl + h * p.o_sh;
  float *lse = p.lse ? p.lse + ((int64_t)b * p.Lq + row) * p.H + h : nullptr;
  const int base = p.prefix[item], n = (p.prefix[item + 1] - base) / p.Hkv, total = p.prefix[p.B * p.blocks];
  if (row >= count || n == 0) {
    if (piece == 0) {
      for (int e = 0; e < 4; ++e) out[d + e] = __float2bfloat16_rn(0.f);
      if (lse && d == 0) *lse = -INFINITY;
    }
    return;
  }
  const int per = max(p.min_steps, (total + p.ctas - 1) / p.ctas);
  const int first = base + kvh * n;
  const int c0 = first / per, c1 = (first + n - 1) / per;
  if (c0 == c1) return;  // finished by its CTA
  const int64_t slot0 = c0 + (int64_t)item * p.Hkv + kvh;
  const int pieces = c1 - c0 + 1;
  __shared__ float red[kMergeThreads / 32];
  __shared__ __align__(16) float part[kPieces][D];
  __shared__ float sums[kPieces];
  float m = kLowest;
  for (int i = tid; i < pieces; i += kMergeThreads) m = fmaxf(m, p.part_ml[2 * ((slot0 + i) * kRows + r)]);
  m = block_max<kMergeThreads>(m, red);
  float l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = piece; i < pieces; i += kPieces) {
    const int64_t at = (slot0 + i) * kRows + r;
    const float2 ml = *reinterpret_cast<const float2 *>(p.part_ml + 2 * at);
    const float4 x = *reinterpret_cast<const float4 *>(p.part_o + at * D + d);
    const float s = tc::ex2(ml.x - m);
    l = fmaf(ml.y, s, l);
    o.x = fmaf(x.x, s, o.x); o.y = fmaf(x.y, s, o.y); o.z = fmaf(x.z, s, o.z); o.w = fmaf(x.w, s, o.w);
  }
  *reinterpret_cast<float4 *>(&part[piece][d]) = o;
  if (d == 0) sums[piece] = l;
  __syncthreads();
  l = 0.f;
#pragma unroll
  for (int i = 0; i < kPieces; ++i) l += sums[i];
  const float inv = l == 0.f ? 0.f : 1.f / l;
  for (int i = tid; i < D; i += kMergeThreads) {
    float x = 0.f;
#pragma unroll
    for (int k = 0; k < kPieces; ++k) x += part[k][i];
    out[i] = __float2bfloat16_rn(x * inv);
  }
  if (lse && tid == 0) *lse = l == 0.f ? -INFINITY : m * kLn2 + logf(l);
}

// ---- host -----------------------------------------------------------------------------------

constexpr int kSms = 148;

template <int FMT, int D, int NT>
struct Shape;  // granules of a step, warps of a CTA, stages of a warp's ring, CTAs of an SM
template <> struct Shape<FPX_PAGES_INT4, 128, 1> { static constexpr int kGranules = 2, kWarps = 4, kStages = 2, kOcc = 4; };
template <> struct Shape<FPX_PAGES_INT4, 128, 2> { static constexpr int kGranules = 2, kWarps = 4, kStages = 3, kOcc = 3; };
template <> struct Shape<FPX_PAGES_INT4, 256, 1> { static constexpr int kGranules = 2, kWarps = 4, kStages = 2, kOcc = 2; };
template <> struct Shape<FPX_PAGES_BF16, 128, 1> { static constexpr int kGranules = 1, kWarps = 4, kStages = 2, kOcc = 3; };
template <> struct Shape<FPX_PAGES_BF16, 128, 2> { static constexpr int kGranules = 1, kWarps = 4, kStages = 2, kOcc = 3; };
template <> struct Shape<FPX_PAGES_BF16, 256, 1> { static constexpr int kGranules = 1, kWarps = 4, kStages = 3, kOcc = 1; };

struct Layout {
  int nt, blocks, ctas, rows;
  size_t prefix, ml, bytes;
  int64_t units;
};
static size_t up256(size_t x) { return (x + 255) & ~size_t(255); }

template <int FMT, int D, int NT>
constexpr int grid_ctas() {
  return kSms * Shape<FMT, D, NT>::kOcc;
}

// Column tiles: two where one would leave rows over, except at head dim 256 (registers).
static Layout layout_of(int format, int B, int Lq, int H, int Hkv, int d) {
  Layout w{};
  const int64_t rows = (int64_t)Lq * (H / Hkv);
  w.nt = d == 128 && rows > 8 ? 2 : 1;
  w.rows = 8 * w.nt;
  w.blocks = (int)((rows + w.rows - 1) / w.rows);
  if (format == FPX_PAGES_INT4)
    w.ctas = d == 256 ? grid_ctas<FPX_PAGES_INT4, 256, 1>()
                      : w.nt == 1 ? grid_ctas<FPX_PAGES_INT4, 128, 1>() : grid_ctas<FPX_PAGES_INT4, 128, 2>();
  else
    w.ctas = d == 256 ? grid_ctas<FPX_PAGES_BF16, 256, 1>()
                      : w.nt == 1 ? grid_ctas<FPX_PAGES_BF16, 128, 1>() : grid_ctas<FPX_PAGES_BF16, 128, 2>();
  w.units = (int64_t)B * w.blocks * Hkv;
  w.prefix = up256(((size_t)B * w.blocks + 1) * sizeof(int));
  w.ml = up256((size_t)(w.ctas + w.units) * w.rows * 2 * sizeof(float));
  w.bytes = w.prefix + w.ml + (size_t)(w.ctas + w.units) * w.rows * d * sizeof(float);
  return w;
}

template <int FMT, int D, int NT>
static int launch(PagedDecodeParams &p, const Layout &w, cudaStream_t stream) {
  using S = Shape<FMT, D, NT>;
  using Smem = PagedSmem<FMT, D, NT, S::kGranules, S::kWarps, S::kStages>;
  static_assert(sizeof(Smem) <= 227 * 1024, "shared memory of one CTA");
  const auto kernel = paged_decode_kernel<FMT, D, NT, S::kGranules, S::kWarps, S::kStages, S::kOcc>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Smem)) != cudaSuccess)
    return FPX_ERR_CUDA;
  p.min_steps = S::kWarps;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(w.ctas);
  cfg.blockDim = dim3(32 * S::kWarps);
  cfg.dynamicSmemBytes = sizeof(Smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, p) != cudaSuccess) return FPX_ERR_CUDA;
  cfg.gridDim = dim3((unsigned)w.units, w.rows);
  cfg.blockDim = dim3(kMergeThreads);
  cfg.dynamicSmemBytes = 0;
  if (cudaLaunchKernelEx(&cfg, paged_merge_kernel<D, NT>, p) != cudaSuccess) return FPX_ERR_CUDA;
  return FPX_OK;
}

static bool decode_sizes_ok(int B, int Lq, int H, int Hkv) {
  return B > 0 && Lq > 0 && Lq <= 64 && H > 0 && Hkv > 0 && H % Hkv == 0 && H / Hkv <= 16 && Hkv <= 65535 &&
         (int64_t)B * Lq * H <= (1 << 24);
}

}  // namespace fpx

using namespace fpx;

extern "C" size_t fpx_paged_decode_workspace_bytes(int format, int B, int Lq, int H, int Hkv, int d) {
  if ((format != FPX_PAGES_BF16 && format != FPX_PAGES_INT4) || (d != 128 && d != 256) || !decode_sizes_ok(B, Lq, H, Hkv))
    return 0;
  return layout_of(format, B, Lq, H, Hkv, d).bytes;
}

extern "C" int fpx_paged_decode_attention(int format, const void *q, int64_t q_sb, int64_t q_sl, int64_t q_sh, int B,
                                          int Lq, int H, int Hkv, int d, double scale, const void *pool, int pages,
                                          int page_size, const int32_t *table, int64_t table_stride, int max_pages,
                                          const int32_t *starts, const int32_t *counts, void *out, int64_t o_sb,
                                          int64_t o_sl, int64_t o_sh, float *lse, void *workspace,
                                          size_t workspace_bytes, fpx_stream_t stream) {
  FPX_BIND(stream);
  if (!q || !out || B <= 0 || Lq <= 0 || H <= 0 || Hkv <= 0) return FPX_ERR_INVALID;
  PagedDecodeParams p{};
  const int rc = make_page_view(&p.pv, format, pool, pages, page_size, table, table_stride, max_pages, starts, counts,
                                Hkv, d);
  if (rc) return rc;
  if (H % Hkv) return FPX_ERR_SHAPE;
  if (!decode_sizes_ok(B, Lq, H, Hkv)) return FPX_ERR_UNSUPPORTED;
  const RowStrides qs(q_sb, q_sl, q_sh, B, Lq, H);
  if ((reinterpret_cast<uintptr_t>(q) & 15) || !qs.multiples_of(8)) return FPX_ERR_SHAPE;
  const Layout w = layout_of(format, B, Lq, H, Hkv, d);
  if (!workspace || workspace_bytes < w.bytes || (reinterpret_cast<uintptr_t>(workspace) & 15)) return FPX_ERR_WORKSPACE;
  p.q = static_cast<const __nv_bfloat16 *>(q); p.q_sb = qs.b; p.q_sl = qs.l; p.q_sh = qs.h;
  p.out = static_cast<__nv_bfloat16 *>(out); p.o_sb = o_sb; p.o_sl = o_sl; p.o_sh = o_sh;
  p.lse = lse;
  p.B = B; p.Lq = Lq; p.H = H; p.Hkv = Hkv; p.group = H / Hkv; p.blocks = w.blocks;
  p.scale_log2 = (float)scale * kLog2e;
  p.ctas = w.ctas;
  // 32-bit counts of steps: what the table could name in all
  if ((int64_t)B * w.blocks * Hkv * ((int64_t)max_pages << p.pv.page_shift) > 0x7fffffff - (1 << 24))
    return FPX_ERR_UNSUPPORTED;
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  p.prefix = reinterpret_cast<int *>(ws);
  p.part_ml = reinterpret_cast<float *>(ws + w.prefix);
  p.part_o = reinterpret_cast<float *>(ws + w.prefix + w.ml);
  if (format == FPX_PAGES_INT4) {
    if (d == 256) return launch<FPX_PAGES_INT4, 256, 1>(p, w, stream);
    return w.nt == 1 ? launch<FPX_PAGES_INT4, 128, 1>(p, w, stream) : launch<FPX_PAGES_INT4, 128, 2>(p, w, stream);
  }
  if (d == 256) return launch<FPX_PAGES_BF16, 256, 1>(p, w, stream);
  return w.nt == 1 ? launch<FPX_PAGES_BF16, 128, 1>(p, w, stream) : launch<FPX_PAGES_BF16, 128, 2>(p, w, stream);
}
