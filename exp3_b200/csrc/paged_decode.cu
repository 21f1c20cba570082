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
//   K: a nibble alone in a half, n or 16 n in place, is the fp16 number n 2^-24 or n 2^-20
//      (subnormal, exact in the product): one mask a pair of codes, one shift for two pairs. The
//      query's dims of the latter are divided by 16. The offset -8 sum(q) comes from one more
//      product with the groups' scales, and a group's scale multiplies the group's sum.
//   V: codes become the fp16 n - 8 (two logic operations and one exact fma a pair); the scales
//      r < 2 multiply the probabilities, in fp16 (11 bits: its rounding stays below the bf16 of the
//      output; kLift keeps small ones off the subnormals). The row exponent 2^e joins the logit: u = exp2(s + e - m) <=
//      2^14 whatever the values' size, and the sum of weights takes u 2^-e (is_far: where e is large, 2^s itself).
//   bf16 pages: P is split in two bf16 terms, so that it does not round before the output does.
//
// Work is split evenly over the CTAs of one launch, whatever the sequences' lengths: the
// steps (one or two granules of 16 tokens) of all (sequence, row block, KV head) units lie end to
// end, each CTA takes an equal run of them, and its four warps every fourth step, each through its own
// ring of bulk copies (no barrier between warps inside a unit). A unit inside one CTA is
// finished there; the pieces of the others are merged in CTA order by the second launch, so
// results do not depend on timing.
//
// More than 16 columns of int4 pages: paged_decode_tc.cu, where wide_units below says so.
#include "paged_decode.cuh"

namespace fpx {

FPX_INLINE uint32_t transpose8(uint32_t a) {  // 8 x 8 16-bit matrix, one row of pairs a quad
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// D = A B + C, 16 x 16 by 16 x 8, fp32 sums: fp16 operands, bf16 operands, and fp16 with C = 0.
FPX_INLINE void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
FPX_INLINE void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
FPX_INLINE void mma_f16_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// Shared memory of a CTA. The merge of its warps has memory of its own where that leaves as many CTAs
// on an SM (int4 pages): the next unit's first copies are then under way while a unit is merged.
template <int FMT, int D, int NT, int GS, int W, int ST>
struct PagedSmem {
  struct Merge {
    float o[W][8 * NT][D + 4];  // rows 4 words apart in the banks: the lanes of a store then differ in theirs
    float m[W][8 * NT], l[W][8 * NT];
  };
  static constexpr bool kApart = FMT == FPX_PAGES_INT4;
  static constexpr int kRing = W * ST * GS * Granule<FMT, D>::kBytes;
  alignas(128) uint8_t memory[kApart ? kRing + sizeof(Merge) : kRing > sizeof(Merge) ? kRing : sizeof(Merge)];
  uint64_t full[W][ST];
  Scan<W> scan;
  int abort;
  FPX_INLINE uint8_t *ring(int warp) { return memory + warp * (kRing / W); }
  FPX_INLINE Merge &merge() { return *reinterpret_cast<Merge *>(memory + (kApart ? kRing : 0)); }
};

// The warp's share of a unit: its columns' running reference m, sums l and O^T.
template <int D, int NT>
struct Columns {
  float o[D / 16][NT][4];
  float m[NT][2], l[NT][2];
};

// Raises the reference m where a logit has passed the one that set it by kRaise (always on a first finite logit),
// and rescales what was summed under the old one. Where is_far says so, here or earlier in the part, it takes the sums of the
// step's weights itself and leaves none to w; so that this costs others nothing, such steps all come through here.
template <int FMT, int D, int NT, int GS>
FPX_INLINE void follow(Columns<D, NT> &c, const float (&y)[GS][NT][4], float (&w)[GS][2], bool &far) {
  float top[NT][2];
  bool up = far;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      top[n][e] = fmaxf(y[0][n][e], y[0][n][e + 2]);
#pragma unroll
      for (int h = 1; h < GS; ++h) top[n][e] = tc::fmax3(top[n][e], y[h][n][e], y[h][n][e + 2]);
      up |= top[n][e] > c.m[n][e] + (kLift<FMT> + kRaise<FMT>);
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
      const float m = fmaxf(c.m[n][e], x - kLift<FMT>);
      const float half = tc::ex2(0.5f * (c.m[n][e] - m)), keep = half * half;
      c.m[n][e] = m;
      c.l[n][e] = c.l[n][e] * half * half;  // keep may lie below 2^-126 and this above
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        c.o[i][n][e] *= keep;
        c.o[i][n][e + 2] *= keep;
      }
    }
  if constexpr (FMT == FPX_PAGES_INT4) {
    float least = w[0][0];
#pragma unroll
    for (int h = 0; h < GS; ++h) least = fminf(least, fminf(w[h][0], w[h][1]));
    far = far || __any_sync(0xffffffffu, is_far(least));
    if (!far) return;
#pragma unroll
    for (int h = 0; h < GS; ++h)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float log_w = log2_of(w[h][k]);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) c.l[n][e] += tc::ex2(y[h][n][2 * k + e] - c.m[n][e] + log_w);
        w[h][k] = 0.f;
      }
  }
}

// Query fragments of a unit (B operands of S^T = K Q^T), column n = lane / 4 of each tile.
//
// int4: a query row times a power of two that brings its largest element to 2^14 .. 2^15, in
// fp16: exact but for elements 2^20 times smaller than that. The dims whose codes the product takes
// sixteenfold (the odd nibbles, in place) are divided by 16.
template <int FMT, int D, int NT>
struct Queries {
  uint32_t b[D / 16][NT][2];
  // int4: what the codes' offset adds, -8 times the query, summed over each group, as three bf16 terms: it multiplies
  // the groups' scales in one more product of four groups x (high, middle, low) for every 128 dims
  uint32_t off[FMT == FPX_PAGES_INT4 ? D / 128 : 1][NT][2];
  float scale[NT][2];  // from S^T to log2 units, columns 2 t, 2 t + 1
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
      // largest exponent of the row, from the elements' bits without their sign
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < D / 32; ++j)
#pragma unroll
        for (uint32_t v : {w[j].x, w[j].y, w[j].z, w[j].w}) top = max(top, max((v << 16) & 0x7fff0000u, v & 0x7fff0000u));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int up = top == 0 ? 0 : min(14 + 127 - (int)(top >> 23), 103);  // at least 14 - 128
      const float mul = __uint_as_float((uint32_t)(127 + up) << 23);
      const float back = logit_factor(p.scale_log2, up);
      f.scale[n][0] = __shfl_sync(0xffffffffu, back, 8 * t);
      f.scale[n][1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
#pragma unroll
      for (int J = 0; J < D / 128; ++J) {
        float sum[4];
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
          const int j = 4 * J + jj;
          const uint32_t v[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
          float x[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(v[i] << 16) * mul;
            x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u) * mul;
          }
          // the codes' pairs are (i, i + 4) of a lane's eight dims; odd ones stand sixteenfold
          f.b[2 * j][n][0] = pack_f16(x[0], x[4]);
          f.b[2 * j][n][1] = pack_f16(x[1] * 0.0625f, x[5] * 0.0625f);
          f.b[2 * j + 1][n][0] = pack_f16(x[2], x[6]);
          f.b[2 * j + 1][n][1] = pack_f16(x[3] * 0.0625f, x[7] * 0.0625f);
          float s = ((x[0] + x[4]) + (x[2] + x[6])) + ((x[1] + x[5]) + (x[3] + x[7]));
          s += __shfl_xor_sync(0xffffffffu, s, 1);
          s += __shfl_xor_sync(0xffffffffu, s, 2);
          sum[jj] = s * -0x1p-21f;  // -8 2^-24
        }
        // k = 2 t, 2 t + 1 of the product: groups 2 (t & 1), + 1; terms high (t < 2), middle; k + 8: low, none
        const float x0 = t & 1 ? sum[2] : sum[0], x1 = t & 1 ? sum[3] : sum[1];
        const float h0 = __bfloat162float(__float2bfloat16_rn(x0)), h1 = __bfloat162float(__float2bfloat16_rn(x1));
        const float m0 = __bfloat162float(__float2bfloat16_rn(x0 - h0)), m1 = __bfloat162float(__float2bfloat16_rn(x1 - h1));
        f.off[J][n][0] = t < 2 ? pack_bf16(h0, h1) : pack_bf16(m0, m1);
        f.off[J][n][1] = t < 2 ? pack_bf16(x0 - h0 - m0, x1 - h1 - m1) : 0u;
      }
    } else {
      f.scale[n][0] = f.scale[n][1] = p.scale_log2;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        f.b[kk][n][0] = live ? *reinterpret_cast<const uint32_t *>(q + 16 * kk + 2 * t) : 0u;
        f.b[kk][n][1] = live ? *reinterpret_cast<const uint32_t *>(q + 16 * kk + 8 + 2 * t) : 0u;
      }
    }
  }
}

// Where a lane reads in a granule.
template <int FMT, int D>
struct Lane {
  int g, t;
  int k, ks, v, vs, ve;  // int4: key codes, their scales, value codes, their scales, exponents
  FPX_INLINE explicit Lane(int lane) : g(lane >> 2), t(lane & 3) {
    if constexpr (FMT == FPX_PAGES_INT4) {
      using G = Granule<FMT, D>;
      k = g * (D / 2) + t * 16;
      ks = G::kKScales + g * (D / 16);
      v = G::kVCodes + v_chunk(2 * t, 0, g);
      vs = G::kVScales + t * (D / 8);
      ve = G::kVExps + 2 * g;
    }
  }
};

// S^T of one granule: y[n] = keys (g, g + 8) x columns (2 t, 2 t + 1), without the scale.
template <int FMT, int D, int NT>
FPX_INLINE void scores(float (&y)[NT][4], const Queries<FMT, D, NT> &f, uint32_t gran, const Lane<FMT, D> &at, int lane) {
#pragma unroll
  for (int n = 0; n < NT; ++n) y[n][0] = y[n][1] = y[n][2] = y[n][3] = 0.f;
  if constexpr (FMT == FPX_PAGES_INT4) {
#pragma unroll
    for (int J = 0; J < D / 128; ++J) {
      const uint4 ka = lds128(gran + at.k + J * 64), kb = lds128(gran + at.k + J * 64 + 8 * (D / 2));
      const uint2 sa = lds64(gran + at.ks + 8 * J), sb = lds64(gran + at.ks + 8 * J + 8 * (D / 16));
      const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
      const uint32_t xa = at.t & 1 ? sa.y : sa.x, xb = at.t & 1 ? sb.y : sb.x;
      const uint32_t s4[4] = {xa, xb, xa, xb};
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_bf16(y[n], s4, f.off[J][n][0], f.off[J][n][1]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t lo = 0x000f000fu, hi = 0x00f000f0u;
        const uint32_t va = wa[j] >> 8, vb = wb[j] >> 8;
        const uint32_t a0[4] = {wa[j] & lo, wb[j] & lo, wa[j] & hi, wb[j] & hi};
        const uint32_t a1[4] = {va & lo, vb & lo, va & hi, vb & hi};
        const uint32_t ua = j < 2 ? sa.x : sa.y, ub = j < 2 ? sb.x : sb.y;
        const float fa = __uint_as_float(j & 1 ? ua & 0xffff0000u : ua << 16);
        const float fb = __uint_as_float(j & 1 ? ub & 0xffff0000u : ub << 16);
        const int gr = 4 * J + j;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float acc[4];
          mma_f16_first(acc, a0, f.b[2 * gr][n][0], f.b[2 * gr][n][1]);
          mma_f16(acc, a1, f.b[2 * gr + 1][n][0], f.b[2 * gr + 1][n][1]);
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
    for (int kk = 0; kk < D / 16; ++kk) {
      uint32_t a[4];
      ldmatrix_x4(a[0], a[1], a[2], a[3], gran + r * Granule<FMT, D>::kRow + (((2 * kk + hi) ^ (r & 7)) << 4));
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_bf16(y[n], a, f.b[kk][n][0], f.b[kk][n][1]);
    }
  }
}

// The probabilities of one granule as the B operands of O^T = V^T P^T, keys along the product.
template <int FMT, int NT>
struct Weights {
  uint32_t b[NT][2];
  uint32_t low[FMT == FPX_PAGES_BF16 ? NT : 1][2];  // bf16: what b's rounding left
};
template <int FMT, int NT>
FPX_INLINE void transpose_weights(Weights<FMT, NT> &p, const float (&u)[NT][4]) {
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float x0 = u[n][2 * e], x1 = u[n][2 * e + 1];
      if constexpr (FMT == FPX_PAGES_INT4) {
        p.b[n][e] = transpose8(pack_f16(x0, x1));
      } else {
        const uint32_t h = pack_bf16(x0, x1);
        p.b[n][e] = transpose8(h);
        p.low[n][e] = transpose8(pack_bf16(x0 - __uint_as_float(h << 16), x1 - __uint_as_float(h & 0xffff0000u)));
      }
    }
}

// O^T += V^T P^T of one granule.
template <int FMT, int D, int NT>
FPX_INLINE void values(Columns<D, NT> &c, const Weights<FMT, NT> &p, uint32_t gran, const Lane<FMT, D> &at, int lane) {
  if constexpr (FMT == FPX_PAGES_INT4) {
#pragma unroll
    for (int J = 0; J < D / 128; ++J) {
      // token pairs t and t + 4: their chunks' places differ by 512 bytes
      const uint4 va = lds128(gran + at.v + 1024 * J), vb = lds128(gran + at.v + 1024 * J + 512);
      const uint4 ra = lds128(gran + at.vs + 16 * J), rb = lds128(gran + at.vs + 16 * J + 4 * (D / 8));
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
          const uint32_t b0 = hmul2u(p.b[n][0], r0[j]), b1 = hmul2u(p.b[n][1], r1[j]);
          mma_f16(c.o[i][n], a0, b0, b1);
          mma_f16(c.o[i + 1][n], a1, b0, b1);
        }
      }
    }
  } else {
    using G = Granule<FMT, D>;
    const int r = (lane & 7) + ((lane >> 4) << 3), hi = (lane >> 3) & 1;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      uint32_t a[4];
      ldmatrix_x4_trans(a[0], a[1], a[2], a[3], gran + r * G::kRow + 2 * D + (((2 * i + hi) ^ (r & 7)) << 4));
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mma_bf16(c.o[i][n], a, p.b[n][0], p.b[n][1]);
        mma_bf16(c.o[i][n], a, p.low[n][0], p.low[n][1]);
      }
    }
  }
}

// Tokens of a granule from `have` on are not there (no row sees them, or their page is missing), and their memory
// may hold anything: their values become zero in the stage, bf16 rows themselves, int4 by scales and exponents.
template <int FMT, int D>
FPX_INLINE void blank(uint32_t gran, int have, int lane) {
  using G = Granule<FMT, D>;
  if constexpr (FMT == FPX_PAGES_INT4) {
    for (int i = lane; i < kGranule * (D / 32 + 1); i += 32) {
      const int token = i % kGranule, group = i / kGranule;
      const int place = group < D / 32 ? G::kVScales + (((token >> 1) * (D / 32) + group) * 2 + (token & 1)) * 2 : G::kVExps + 2 * token;
      if (token >= have) asm volatile("st.shared.u16 [%0], %1;" ::"r"(gran + place), "h"((uint16_t)0) : "memory");
    }
  } else {
    for (int i = lane; i < kGranule * (D / 8); i += 32) {
      const int token = i / (D / 8);
      if (token >= have)
        asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(gran + token * G::kRow + 2 * D + 16 * (i % (D / 8))), "r"(0)
                     : "memory");
    }
  }
}

FPX_INLINE void sts16(uint32_t a, uint16_t v) { asm volatile("st.shared.u16 [%0], %1;" ::"r"(a), "h"(v) : "memory"); }
FPX_INLINE bool no_number_f16(uint32_t x) { return (x & 0x7c00u) == 0x7c00u; }
FPX_INLINE bool no_number_bf16(uint32_t x) { return (x & 0x7f80u) == 0x7f80u; }

// Tokens `first` .. have - 1 of a granule are seen by some columns and not by others, whose probability 0 times an
// infinity or a NaN in the value would be NaN. Such values become zero in the stage, and the sums of the columns that see them
// (limit: the first unseen key) NaN here. key0: the granule's first key.
template <int FMT, int D, int NT>
FPX_INLINE void settle(Columns<D, NT> &c, const int (&limit)[NT][2], uint32_t gran, int key0, int first, int have, int lane) {
  using G = Granule<FMT, D>;
  const int g = lane >> 2;
  bool any = false;
  if constexpr (FMT == FPX_PAGES_INT4) {
    // a group of a row: its scale says so
    auto place = [&](int token, int group) { return gran + G::kVScales + (((token >> 1) * (D / 32) + group) * 2 + (token & 1)) * 2; };
    for (int i = lane; i < kGranule * (D / 32); i += 32) {
      const int token = i % kGranule;
      any |= token >= first && token < have && no_number_f16(lds16(place(token, i / kGranule)));
    }
    if (!__any_sync(0xffffffffu, any)) return;
#pragma unroll 1
    for (int token = first; token < have; ++token)
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        if (!no_number_f16(lds16(place(token, j)))) continue;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (key0 + token < limit[n][e])
              c.o[2 * j][n][e] = c.o[2 * j][n][e + 2] = c.o[2 * j + 1][n][e] = c.o[2 * j + 1][n][e + 2] = __uint_as_float(0x7fffffffu);
      }
    __syncwarp();
    for (int i = lane; i < kGranule * (D / 32); i += 32) {
      const int token = i % kGranule;
      const uint32_t a = place(token, i / kGranule);
      if (token >= first && token < have && no_number_f16(lds16(a))) sts16(a, 0);
    }
  } else {
    auto place = [&](int token, int chunk) { return gran + token * G::kRow + 2 * D + ((chunk ^ (token & 7)) << 4); };
    for (int i = lane + first * (D / 8); i < have * (D / 8); i += 32) {
      const uint4 w = lds128(place(i / (D / 8), i % (D / 8)));
      for (uint32_t x : {w.x, w.y, w.z, w.w}) any |= no_number_bf16(x) || no_number_bf16(x >> 16);
    }
    if (!__any_sync(0xffffffffu, any)) return;
#pragma unroll 1
    for (int token = first; token < have; ++token)
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {  // dims 16 i + 8 k + g
          const uint32_t x = lds16(place(token, 2 * i + k) + 2 * g);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (no_number_bf16(x) && key0 + token < limit[n][e]) c.o[i][n][e + 2 * k] = __uint_as_float(0x7fffffffu);
        }
    __syncwarp();
    for (int i = lane + first * (D / 8); i < have * (D / 8); i += 32) {
      const uint32_t a = place(i / (D / 8), i % (D / 8));
      for (int d = 0; d < 8; ++d)
        if (no_number_bf16(lds16(a + 2 * d))) sts16(a + 2 * d, 0);
    }
  }
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
  if (lane < ST) tc::mbar_init(&sh.full[warp][lane], 1);
  if (tid == 0) sh.abort = 0;
  tc::fence_barrier_init();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  Walk<NT, GS> u;
  if (!u.begin(p, sh.scan, tid)) return;
  __syncthreads();  // the ring's barriers are set

  const Lane<FMT, D> at(lane);
  uint8_t *const ring_bytes = sh.ring(warp);
  const uint32_t ring = smem_u32(ring_bytes);

  int &b = u.b, &rb = u.rb, &kvh = u.kvh, &start = u.start, &rows = u.rows, &seen = u.seen, &n_steps = u.n_steps, &g0 = u.g0,
      &g1 = u.g1, &item = u.item;
  // Ring: step g0 + warp + W i of the part goes into the next stage. A lane works out where one of the
  // next 32 steps lies (16 where each granule has a page of its own).
  const bool paired = GS == 2 && p.pv.page_shift == 0;
  int todo = 0, sent = 0, put = 0, get = 0;  // stages to fill and to read next
  uint32_t phase = 0, dead = 0;              // a bit a stage: parity of its next wait; GS bits a stage: missing granules
  uint32_t here = 0;                         // bit i: the page of lane i's granules exists
  uint64_t source = 0;
  bool stopped = false;
  auto issue = [&]() {
    const int per_block = paired ? 16 : 32;
    const int slot = sent & (per_block - 1);
    if (slot == 0) {
      const int step = g0 + warp + W * (sent + (paired ? lane >> 1 : lane));
      const int granule = GS * step + (paired ? lane & 1 : 0);
      const int last_page = (seen - 1) >> (p.pv.page_shift + 4);
      const int at_page = granule >> p.pv.page_shift;
      const int page = p.pv.table[(int64_t)b * p.pv.table_stride + min(at_page, last_page)];
      const bool wanted = at_page <= last_page && step < g1, ok = (unsigned)page < (unsigned)p.pv.pages;
      if (wanted && !ok) p.pv.fail();
      here = __ballot_sync(0xffffffffu, wanted && ok);
      source = reinterpret_cast<uint64_t>(p.pv.pool) + (int64_t)kvh * p.pv.head_bytes +
               (int64_t)(ok ? page : 0) * p.pv.page_bytes + (granule & ((1 << p.pv.page_shift) - 1)) * G::kBytes;
    }
    const uint64_t src = __shfl_sync(0xffffffffu, source, paired ? 2 * slot : slot);
    uint64_t *bar = &sh.full[warp][put];
    uint8_t *dst = ring_bytes + put * kBytes;
    dead &= ~(kAll << (GS * put));
    if (!paired) {
      if (!((here >> slot) & 1)) dead |= kAll << (GS * put);
      if (lane == 0) {
        tc::mbar_expect_tx(bar, kBytes);
        bulk_load(dst, reinterpret_cast<const void *>(src), kBytes, bar);
      }
    } else {  // the second granule of a sequence's last step may not exist
      const uint64_t src2 = __shfl_sync(0xffffffffu, source, 2 * slot + 1);
      const uint32_t two = (here >> (2 * slot)) & 3u;
      dead |= (two ^ 3u) << (GS * put);
      if (lane == 0) {
        tc::mbar_expect_tx(bar, two & 2 ? 2 * G::kBytes : G::kBytes);
        bulk_load(dst, reinterpret_cast<const void *>(src), G::kBytes, bar);
        if (two & 2) bulk_load(dst + G::kBytes, reinterpret_cast<const void *>(src2), G::kBytes, bar);
      }
    }
    put = put + 1 == ST ? 0 : put + 1;
    ++sent;
  };
  auto arrived = [&](int stage) {  // the copy that was put there last
    if (!tc::mbar_wait_warp(&sh.full[warp][stage], (phase >> stage) & 1, &sh.abort)) {
      stopped = true;  // it did not arrive: report it and let the launch end
      if (lane == 0 && p.error) atomicMax(p.error, FPX_DEVICE_WAIT);
      return false;
    }
    phase ^= 1u << stage;
    return true;
  };
  auto begin = [&]() {  // the part's first copy; the others follow once its queries are loaded, so that
    todo = g1 - g0 > warp ? (g1 - g0 - warp + W - 1) / W : 0;  // every warp's first is early in the queue
    sent = 0;
    if (todo > 0 && !stopped) issue();
  };
  if (p.whole) {
    u.whole(p);
    // rows that see nothing: padding, and inactive sequences
    for (int i = max(0, rows - rb * kRows) * (D / 4) + tid; i < min(kRows, p.Lq * p.group - rb * kRows) * (D / 4); i += kThreads) {
      const int r = rb * kRows + i / (D / 4), row = r / p.group, h = kvh * p.group + r % p.group, d = 4 * (i % (D / 4));
      __nv_bfloat16 *out = p.out + b * p.o_sb + row * p.o_sl + h * p.o_sh + d;
      out[0] = out[1] = out[2] = out[3] = __float2bfloat16_rn(0.f);
      if (p.lse && d == 0) p.lse[((int64_t)b * p.Lq + row) * p.H + h] = -INFINITY;
    }
    if (n_steps == 0) return;
  } else if (!u.find(p)) {
    return;
  }
  begin();
  for (;;) {
    const int row0 = rb * kRows;
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
    while (sent < min(todo, ST) && !stopped) issue();
    Columns<D, NT> c;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      c.m[n][0] = c.m[n][1] = kLowest;
      c.l[n][0] = c.l[n][1] = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) c.o[i][n][0] = c.o[i][n][1] = c.o[i][n][2] = c.o[i][n][3] = 0.f;
    }
    // Software pipeline: the next step's scores share a block with this step's values, so that each
    // covers the other's latencies.
    float y[GS][NT][4];
    Weights<FMT, NT> pw[GS];
    bool far = false;  // as is_far has it
    auto weigh = [&](int i) {  // from the scores of step i, which lies in stage `get`, to its probabilities
      const uint32_t stage = ring + get * kBytes;
      const int key0 = (g0 + warp + W * i) * kStep;
      const uint32_t gone = (dead >> (GS * get)) & kAll;
      const bool edge = key0 + kStep > least || gone;
      if (edge) {
#pragma unroll
        for (int h = 0; h < GS; ++h) {
          const int have = (gone >> h) & 1 ? 0 : seen - key0 - kGranule * h;
          if (have < kGranule) blank<FMT, D>(stage + h * G::kBytes, have, lane);
          const int first = max(least - key0 - kGranule * h, 0), last = min(have, kGranule);
          if (first < last) settle<FMT, D, NT>(c, limit, stage + h * G::kBytes, key0 + kGranule * h, first, last, lane);
        }
        tc::fence_proxy_async();  // before the next copy into this stage
        __syncwarp();
      }
      float w[GS][2];  // 2^(kSumLift - e) of the lane's two keys
#pragma unroll
      for (int h = 0; h < GS; ++h) {
        float e[2] = {0.f, 0.f};  // row exponents of the two keys' values
        w[h][0] = w[h][1] = kSumUnit;
        if (FMT == FPX_PAGES_INT4) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            e[k] = __uint_as_float(lds16(stage + h * G::kBytes + at.ve + 16 * k) << 16);
            w[h][k] = tc::ex2(kSumLift - e[k]);
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int k = 0; k < 4; ++k) y[h][n][k] = fmaf(y[h][n][k], f.scale[n][k & 1], e[k >> 1]);
      }
      if (edge) {
#pragma unroll
        for (int h = 0; h < GS; ++h)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (((gone >> h) & 1) || key0 + kGranule * h + g + 8 * (k >> 1) >= limit[n][k & 1]) y[h][n][k] = -INFINITY;
      }
      follow<FMT, D, NT, GS>(c, y, w, far);
#pragma unroll
      for (int h = 0; h < GS; ++h) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int k = 0; k < 4; ++k) y[h][n][k] = tc::ex2(y[h][n][k] - c.m[n][k & 1]);
          c.l[n][0] = fmaf(y[h][n][0], w[h][0], fmaf(y[h][n][2], w[h][1], c.l[n][0]));
          c.l[n][1] = fmaf(y[h][n][1], w[h][0], fmaf(y[h][n][3], w[h][1], c.l[n][1]));
        }
        transpose_weights<FMT, NT>(pw[h], y[h]);
      }
    };
    if (todo > 0 && !stopped && arrived(get)) {
#pragma unroll
      for (int h = 0; h < GS; ++h) scores<FMT, D, NT>(y[h], f, ring + get * kBytes + h * G::kBytes, at, lane);
      for (int i = 0;; ++i) {
        weigh(i);
        if (i + 1 == todo) break;
        const int after = get + 1 == ST ? 0 : get + 1;
        if (!arrived(after)) break;
        const uint32_t stage = ring + get * kBytes, next = ring + after * kBytes;
#pragma unroll
        for (int h = 0; h < GS; ++h) {
          scores<FMT, D, NT>(y[h], f, next + h * G::kBytes, at, lane);
          values<FMT, D, NT>(c, pw[h], stage + h * G::kBytes, at, lane);
        }
        get = after;
        if (sent < todo) {
          __syncwarp();  // every lane has read the stage
          issue();
        }
      }
      if (!stopped) {
#pragma unroll
        for (int h = 0; h < GS; ++h) values<FMT, D, NT>(c, pw[h], ring + get * kBytes + h * G::kBytes, at, lane);
        get = get + 1 == ST ? 0 : get + 1;
      }
    }
    if (stopped)  // copies still in flight end before this memory is used again, or this long later
      for (int st = 0; st < ST; ++st) {
        const long long from = clock64();
        while (!tc::mbar_test(&sh.full[warp][st], (phase >> st) & 1) && clock64() - from < tc::kWaitCycles / 8) {
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
    const bool whole = g0 == 0 && g1 == n_steps;
    const int64_t slot = blockIdx.x + (int64_t)item * p.Hkv + kvh;
    const int mb = b, mkvh = kvh, mrows = rows;
    const bool more = u.find(p);
    if (Smem::kApart) {
      if (more) begin();
    } else {
      __syncthreads();  // every warp has read its last step
    }
    typename Smem::Merge &merge = sh.merge();
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = 8 * n + 2 * t + e;
        if (g == 0) {
          merge.m[warp][col] = c.m[n][e];
          merge.l[warp][col] = c.l[n][e];
        }
        if constexpr (FMT == FPX_PAGES_INT4) {  // the value codes' layout gives a lane four neighbouring dims over two tiles
#pragma unroll
          for (int i = 0; i < D / 16; i += 2)
            *reinterpret_cast<float4 *>(&merge.o[warp][col][16 * i + 4 * g]) =
                make_float4(c.o[i][n][e], c.o[i][n][e + 2], c.o[i + 1][n][e], c.o[i + 1][n][e + 2]);
        } else {
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            merge.o[warp][col][16 * i + g] = c.o[i][n][e];
            merge.o[warp][col][16 * i + 8 + g] = c.o[i][n][e + 2];
          }
        }
      }
    __syncthreads();
    constexpr int kQuads = D / 4;
    for (int i = tid; i < kRows * kQuads; i += kThreads) {
      const int r = i / kQuads, d = 4 * (i % kQuads);
      if (row0 + r >= mrows) break;
      float m = merge.m[0][r], l = 0.f;
#pragma unroll
      for (int w = 1; w < W; ++w) m = fmaxf(m, merge.m[w][r]);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float half = tc::ex2(0.5f * (merge.m[w][r] - m)), s = half * half;
        const float4 x = *reinterpret_cast<const float4 *>(&merge.o[w][r][d]);
        l = fmaf(merge.l[w][r] * half, half, l);
        o.x = fmaf(x.x, s, o.x); o.y = fmaf(x.y, s, o.y); o.z = fmaf(x.z, s, o.z); o.w = fmaf(x.w, s, o.w);
      }
      if (whole) {
        const int row = (row0 + r) / p.group, h = mkvh * p.group + (row0 + r) % p.group;
        const float inv = inverse_sum(l);
        __nv_bfloat16 *out = p.out + mb * p.o_sb + row * p.o_sl + h * p.o_sh + d;
        out[0] = __float2bfloat16_rn(o.x * inv); out[1] = __float2bfloat16_rn(o.y * inv);
        out[2] = __float2bfloat16_rn(o.z * inv); out[3] = __float2bfloat16_rn(o.w * inv);
        if (p.lse && d == 0) p.lse[((int64_t)mb * p.Lq + row) * p.H + h] = log_sum(m, l);
      } else {
        *reinterpret_cast<float4 *>(&p.part_o[(slot * kRows + r) * D + d]) = o;
        if (d == 0) *reinterpret_cast<float2 *>(&p.part_ml[2 * (slot * kRows + r)]) = make_float2(m, l);
      }
    }
    if (!more) return;
    if (!Smem::kApart) tc::fence_proxy_async();  // these accesses come before the next unit's copies
    __syncthreads();
    if (!Smem::kApart) begin();
  }
}

// ---- host -----------------------------------------------------------------------------------

template <int FMT, int D, int NT>
struct Shape;  // granules of a step, warps of a CTA, stages of a warp's ring, CTAs of an SM
template <> struct Shape<FPX_PAGES_INT4, 128, 1> { static constexpr int kGranules = 2, kWarps = 4, kStages = 3, kOcc = 3; };
template <> struct Shape<FPX_PAGES_INT4, 128, 2> { static constexpr int kGranules = 2, kWarps = 4, kStages = 4, kOcc = 2; };
template <> struct Shape<FPX_PAGES_INT4, 256, 1> { static constexpr int kGranules = 2, kWarps = 4, kStages = 2, kOcc = 2; };
template <> struct Shape<FPX_PAGES_BF16, 256, 2> { static constexpr int kGranules = 1, kWarps = 4, kStages = 3, kOcc = 1; };
template <> struct Shape<FPX_PAGES_BF16, 128, 1> { static constexpr int kGranules = 1, kWarps = 4, kStages = 3, kOcc = 2; };
template <> struct Shape<FPX_PAGES_BF16, 128, 2> { static constexpr int kGranules = 1, kWarps = 4, kStages = 3, kOcc = 2; };
template <> struct Shape<FPX_PAGES_BF16, 256, 1> { static constexpr int kGranules = 1, kWarps = 4, kStages = 3, kOcc = 1; };

static size_t up256(size_t x) { return (x + 255) & ~size_t(255); }

template <int FMT, int D, int NT>
constexpr int grid_ctas() {
  return kSms * Shape<FMT, D, NT>::kOcc;
}

// Column tiles of a row block: two where one would leave rows over (16 rows at d = 128: 25.6 us in one block of two
// tiles, 35 in two of one), but one for int4 at d = 256, whose registers two do not fit (16 rows: 59 us, 42 in two blocks).
// Many columns (`wide`): row blocks of 32 or 64 on tcgen05.
static DecodeLayout layout_of(int format, int B, int Lq, int H, int Hkv, int d, bool wide) {
  DecodeLayout w{};
  const int64_t rows = (int64_t)Lq * (H / Hkv);
  w.nt = wide ? (rows > 32 ? 8 : 4) : rows > 8 && !(format == FPX_PAGES_INT4 && d == 256) ? 2 : 1;
  w.rows = 8 * w.nt;
  w.blocks = (int)((rows + w.rows - 1) / w.rows);
  if (wide)
    w.ctas = kSms;
  else if (format == FPX_PAGES_INT4)
    w.ctas = d == 256 ? grid_ctas<FPX_PAGES_INT4, 256, 1>()
                      : (w.nt == 1 ? grid_ctas<FPX_PAGES_INT4, 128, 1>() : grid_ctas<FPX_PAGES_INT4, 128, 2>());
  else
    w.ctas = d == 256 ? (w.nt == 1 ? grid_ctas<FPX_PAGES_BF16, 256, 1>() : grid_ctas<FPX_PAGES_BF16, 256, 2>())
                      : (w.nt == 1 ? grid_ctas<FPX_PAGES_BF16, 128, 1>() : grid_ctas<FPX_PAGES_BF16, 128, 2>());
  w.units = (int64_t)B * w.blocks * Hkv;
  w.prefix = up256(((size_t)B * w.blocks + 1) * sizeof(int));
  w.ml = up256((size_t)(w.ctas + w.units) * w.rows * 2 * sizeof(float));
  w.bytes = w.prefix + w.ml + (size_t)(w.ctas + w.units) * w.rows * d * sizeof(float);
  return w;
}

// Short tables: a CTA a unit, one launch and no workspace. Four KV heads, us in one launch / in two, int4: 1 sequence of 256
// tokens 6.0 / 8.0, 512 7.7 / 8.0, 1024 11.0 / 8.0; 37 sequences 6.8 / 10.2, 8.5 / 14.9, 12.0 / 13.4; bf16: 5.6 / 7.0, 7.5 /
// 7.0, 11.5 / 7.1 and 5.8 / 9.1, 10.1 / 13.3, 15.7 / 19.2. Tables as wide as the sequences: the rule sees the table's width, and where that is more
// than they need (a cache of long slots), short sequences take two launches.
static bool whole_units(const PageView &pv, int64_t units) {
  const int64_t tokens = ((int64_t)pv.max_pages << pv.page_shift) * kGranule;
  return tokens <= (units >= 32 ? 1024 : 512);
}

// Whether the tcgen05 kernel takes int4 pages of more than 16 columns: not where the other one's row blocks are few (w is its
// layout), since it begins a unit 2 to 4 us later. Us, mma.sync / tcgen05: 4 x 65536 tokens, d = 128, 20 columns 33.8 /
// 27.7, 28 35.0 / 27.9, 56 56.2 / 38.9, 448 281 / 175; d = 256, 20 columns 54.5 / 42.7, 64 115 / 59.5; 1 x 8192, 56 columns
// 11.3 / 13.1. Tables of 512 tokens, a CTA a unit: 8 x 4 KV heads, 56 columns 10.9 / 15.7; 32 x 4 23.3 / 17.1. Tables as wide as the sequences, as above.
static bool wide_units(const PageView &pv, const DecodeLayout &w) {
  const int64_t tokens = ((int64_t)pv.max_pages << pv.page_shift) * kGranule;
  return tokens * w.units > 65536 && !(whole_units(pv, w.units) && w.units <= w.ctas);
}
static bool may_be_wide(int format, int Lq, int H, int Hkv) { return format == FPX_PAGES_INT4 && Lq * (H / Hkv) > 16; }

template <int FMT, int D, int NT>
static int launch(PagedDecodeParams &p, const DecodeLayout &w, cudaStream_t stream) {
  using S = Shape<FMT, D, NT>;
  using Smem = PagedSmem<FMT, D, NT, S::kGranules, S::kWarps, S::kStages>;
  static_assert(sizeof(Smem) <= 227 * 1024, "shared memory of one CTA");
  static std::atomic<uint64_t> set{0};
  return launch_decode<D, NT, S::kGranules>(paged_decode_kernel<FMT, D, NT, S::kGranules, S::kWarps, S::kStages, S::kOcc>, set,
                                            32 * S::kWarps, (int)sizeof(Smem), S::kWarps, p, w, stream);
}

static bool decode_sizes_ok(int B, int Lq, int H, int Hkv) {
  return B > 0 && Lq > 0 && Lq <= FPX_PAGED_MAX_ROWS && H > 0 && Hkv > 0 && H % Hkv == 0 && H / Hkv <= 16 && Hkv <= 65535 &&
         (int64_t)B * Lq * H <= (1 << 24);
}

}  // namespace fpx

using namespace fpx;

extern "C" size_t fpx_paged_decode_workspace_bytes(int format, int B, int Lq, int H, int Hkv, int d) {
  if ((format != FPX_PAGES_BF16 && format != FPX_PAGES_INT4) || (d != 128 && d != 256) || !decode_sizes_ok(B, Lq, H, Hkv))
    return 0;
  const size_t bytes = layout_of(format, B, Lq, H, Hkv, d, false).bytes;
  return may_be_wide(format, Lq, H, Hkv) ? std::max(bytes, layout_of(format, B, Lq, H, Hkv, d, true).bytes) : bytes;
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
  DecodeLayout w = layout_of(format, B, Lq, H, Hkv, d, false);
  if (may_be_wide(format, Lq, H, Hkv) && wide_units(p.pv, w)) w = layout_of(format, B, Lq, H, Hkv, d, true);
  p.whole = whole_units(p.pv, w.units);
  if (!p.whole && (!workspace || workspace_bytes < w.bytes || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return FPX_ERR_WORKSPACE;
  p.q = static_cast<const __nv_bfloat16 *>(q); p.q_sb = qs.b; p.q_sl = qs.l; p.q_sh = qs.h;
  p.out = static_cast<__nv_bfloat16 *>(out); p.o_sb = o_sb; p.o_sl = o_sl; p.o_sh = o_sh;
  p.lse = lse;
  p.error = device_error_word();
  p.B = B; p.Lq = Lq; p.H = H; p.Hkv = Hkv; p.group = H / Hkv; p.blocks = w.blocks;
  p.scale_log2 = (float)scale * kLog2e;
  // 32-bit counts of steps: what the table could name in all
  if ((int64_t)B * w.blocks * Hkv * (((int64_t)max_pages << p.pv.page_shift) + kPad) > 0x7fffffff - (1 << 24))
    return FPX_ERR_UNSUPPORTED;
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  p.prefix = reinterpret_cast<int *>(ws);
  p.part_ml = reinterpret_cast<float *>(ws + w.prefix);
  p.part_o = reinterpret_cast<float *>(ws + w.prefix + w.ml);
  if (format == FPX_PAGES_INT4) {
    if (w.nt > 2) return launch_paged_decode_tc(p, w, d, stream);
    if (d == 256) return launch<FPX_PAGES_INT4, 256, 1>(p, w, stream);
    return w.nt == 1 ? launch<FPX_PAGES_INT4, 128, 1>(p, w, stream) : launch<FPX_PAGES_INT4, 128, 2>(p, w, stream);
  }
  if (d == 256) return w.nt == 1 ? launch<FPX_PAGES_BF16, 256, 1>(p, w, stream) : launch<FPX_PAGES_BF16, 256, 2>(p, w, stream);
  return w.nt == 1 ? launch<FPX_PAGES_BF16, 128, 1>(p, w, stream) : launch<FPX_PAGES_BF16, 128, 2>(p, w, stream);
}
