// Decode attention over 4-bit pages for many query columns (more than 16: drafts of several tokens, wide groups), on the
// tcgen05 tensor core. Same mathematics and split of work as paged_decode.cu; here one pass over the codes serves up to
// 64 columns, where mma.sync's accumulators leave room for 8 or 16.
//
// Per tile of 128 keys, S^T = K Q^T (keys x columns) and O^T += V^T P^T (dims x columns): the codes' side of both
// products is the A operand, and A is read from TMEM. The layout of paged.cuh expands a granule into mma.sync's A
// fragments, which is what tcgen05.st's 16x128b shape stores: rows of the operand are its lanes, pairs along the
// product its columns, so dequantised tiles never pass through shared memory (written and read there they would take
// 2600 of its cycles a tile at d = 256, where HBM takes 1600). Only queries and probabilities, the B operands, do.
//   K: fp16 (n - 8) s 2^-E, E the key's own exponent: 3 + 8 bits, exact down to 2^-30 of the key's largest group. The key is
//      a lane of S^T, so 2^E, the row exponent e and 2^-e are registers of the thread that reads it.
//   V: fp16 (n - 8) r, rounded once; probabilities fp16, at most 2^14. Both roundings stay below the output's bf16.
//
// A CTA: warps 0-3 and 4-7 do the softmax of half the columns each (thread = key; neither half waits for the other), warps
// 8-11 expand keys, warps 12-15 values (warp = 32 dims of each 128, the lanes that it may write), warp 16 issues the bulk
// copies, warps 17 and 18 the products. The next tile's scores are computed while this one's softmax runs.
//
// Measured (4 sequences of 65536 tokens, one KV head, us of one call): d = 128, 28 columns 27.9, 56 columns 38.8, 448 columns 175; d =
// 256, 20 columns 42.7, 64 columns 59.4. What bounds it: the latency of the softmax warps (2000 to 2500 cycles a tile at d =
// 128, where a product takes the tensor core 63 cycles whatever its columns and 16 of them 1000), the expansion of values
// (1400, and 2700 at d = 256) and the issue of products (100 to 150 cycles each); 8 us of it begin and merge.
#include "paged_decode.cuh"

namespace fpx {
namespace {

using namespace tc;

constexpr int kTile = 128;            // keys
constexpr int kGs = kTile / kGranule;  // granules of a step
constexpr float kLift4 = kLift<FPX_PAGES_INT4>, kRaise4 = kRaise<FPX_PAGES_INT4>;
constexpr int kTcThreads = 640;  // five warpgroups; one of the last one's warps only makes up its number

// 16 rows (lanes) x 32 columns of TMEM: lane 4 g + t holds rows g and g + 8 of columns t, 4 + t, ..
FPX_INLINE void tmem_st_16x128b_x8(uint32_t taddr, const uint32_t (&u)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
      "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15])
      : "memory");
}
// kind::f16 with fp16 operands, M = 128, fp32 sums; A from TMEM.
constexpr uint32_t idesc_f16(int N, bool b_mn_major) {
  return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// C consecutive fp32 columns of the thread's TMEM lane.
FPX_INLINE void tmem_load(uint32_t taddr, float (&r)[32]) { tmem_ld32(taddr, r); }
FPX_INLINE void tmem_load(uint32_t taddr, float (&r)[16]) {
  uint32_t *u = reinterpret_cast<uint32_t *>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]),
        "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
      : "r"(taddr));
}
FPX_INLINE void tmem_ld8(uint32_t taddr, float (&r)[8]) {
  uint32_t *u = reinterpret_cast<uint32_t *>(r);
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7])
               : "r"(taddr));
}
FPX_INLINE void tmem_st8(uint32_t taddr, const float (&r)[8]) {
  const uint32_t *u = reinterpret_cast<const uint32_t *>(r);
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(u[0]), "r"(u[1]),
               "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
               : "memory");
}
// Folds 16 or 32 columns over the warp: lane n gets column n's (mod 16).
template <int C, typename F>
FPX_INLINE float fold(float (&x)[C], int lane, F f) {
#pragma unroll
  for (int o = C / 2; o; o >>= 1)
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const bool high = lane & o;
      const float give = high ? x[i] : x[i + o], have = high ? x[i + o] : x[i];
      x[i] = f(have, __shfl_xor_sync(0xffffffffu, give, o));
    }
  return C == 16 ? f(x[0], __shfl_xor_sync(0xffffffffu, x[0], 16)) : x[0];
}
// Whether a tile may have keys that are not there, or that some columns see and others do not.
FPX_INLINE bool edge_tile(int step, int seen) { return step * kTile + kTile > seen - FPX_PAGED_MAX_ROWS; }
// Scales that are no numbers as fp16's largest, times whose codes, n - 8 = 0, is zero.
FPX_INLINE uint32_t numbers(uint32_t scales) {
  const __half2 v = __hmin2(*reinterpret_cast<const __half2 *>(&scales), __half2half2(__ushort_as_half(0x7bff)));
  return *reinterpret_cast<const uint32_t *>(&v);
}
FPX_INLINE uint32_t half2_of(float x) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %1;" : "=r"(d) : "f"(x));
  return d;
}

// N columns of a row block; stages of a tile's codes, buffers of expanded keys and values.
template <int D, int N>
struct TcShape {
  static constexpr int kStages = D == 128 ? 6 : 4;
  static constexpr int kKBufs = D == 256 ? 1 : 2, kVBufs = D == 256 && N == 64 ? 1 : 2;
  // TMEM columns: keys, values, two S^T, O^T
  static constexpr uint32_t kK = 0, kV = kKBufs * (D / 2), kS = kV + kVBufs * (D / 2), kO = kS + 2 * N, kEnd = kO + D / 128 * N;
  static_assert(kEnd <= 512, "TMEM");
};

template <int D, int N>
struct alignas(1024) TcSmem {
  static constexpr int ST = TcShape<D, N>::kStages;
  static constexpr int kStage = kGs * Granule<FPX_PAGES_INT4, D>::kBytes;
  uint8_t q[N * D * 2];           // B operand of S^T: rows of 64 halves, 128-byte swizzle, D / 64 of them side by side
  uint8_t pr[2][kTile * 128];     // B operand of O^T: a row a key, its columns in place, 128-byte swizzle
  uint8_t stage[ST][kStage];
  float4 column[N / 2];           // of columns 2 i, 2 i + 1: scales of S, and minus their references
  int limit[N];                   // first key that the column does not see
  int64_t out_at[N];              // element of `out` where its row begins; lse's at
  int lse_at[N];
  float keep[N], by[N], sum[N], red[4][N];  // keep: square root of what a reference's move leaves of the sums
  int4 vote[2][2];                // of each half
  // Of each group and key warp: first key of the edge tiles whose value's group is no number. The
  // products take it as zero, since a probability 0 times it would be NaN; the columns that see it become NaN at the end. By part, in
  // four places: key warps begin a part when the softmax may still have to read of the third part before it, and no earlier one.
  int4 spoilt[4][D / 32];
  int gone[ST];                   // a bit a granule: its page is missing
  uint64_t full[ST], empty[ST], q_ready, k_ready[2], v_ready[2], p_ready[2], s_full[2], s_free[2], pv_done[2], spoilt_ready[4], drain[2];
  Scan<kTcThreads / 32> scan;
  uint32_t tmem;
  int abort;
};

template <int D, int N>
__global__ void __launch_bounds__(kTcThreads, 1) paged_decode_tc_kernel(const __grid_constant__ PagedDecodeParams p) {
  using G = Granule<FPX_PAGES_INT4, D>;
  using S = TcShape<D, N>;
  using Smem = TcSmem<D, N>;
  constexpr int ST = S::kStages, KB = S::kKBufs, VB = S::kVBufs, J = D / 128, C = N / 2;
  extern __shared__ uint8_t smem_raw[];
  Smem &sh = *reinterpret_cast<Smem *>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
  volatile int *abort = &sh.abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  if (tid == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], 16);
    }
    mbar_init(&sh.q_ready, 8);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.k_ready[i], 4);
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.s_free[i], 8);
      mbar_init(&sh.p_ready[i], 8);
      mbar_init(&sh.v_ready[i], 4);
      mbar_init(&sh.pv_done[i], 1);
      mbar_init(&sh.drain[i], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&sh.spoilt_ready[i], 4);
    sh.abort = 0;
    fence_barrier_init();
  }
  if (warp == 16) {
    tmem_alloc(&sh.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  Walk<N / 8, kGs> u;
  bool work = u.begin(p, sh.scan, tid);
  if (p.whole) {
    u.whole(p);
    // rows that see nothing: padding, and inactive sequences
    const int row0 = u.rb * N;
    for (int i = max(0, u.rows - row0) * (D / 4) + tid; i < min(N, p.Lq * p.group - row0) * (D / 4); i += kTcThreads) {
      const int r = row0 + i / (D / 4), row = r / p.group, h = u.kvh * p.group + r % p.group, d = 4 * (i % (D / 4));
      __nv_bfloat16 *out = p.out + u.b * p.o_sb + row * p.o_sl + h * p.o_sh + d;
      out[0] = out[1] = out[2] = out[3] = __float2bfloat16_rn(0.f);
      if (p.lse && d == 0) p.lse[((int64_t)u.b * p.Lq + row) * p.H + h] = -INFINITY;
    }
    work = u.n_steps > 0;
  } else if (work) {
    work = u.find(p);
  }
  // 128 x (128 + 128 + 80 + 80 + 64) registers of the launch's 640 x 96
  if (warp < 8)
    regs_inc<128>();
  else if (warp < 16)
    regs_dec<80>();
  else
    regs_dec<64>();
  int c = 0;  // tiles of this CTA so far: tile c lies in stage c % ST, S^T and P^T buffers c & 1
  int parts = 0;
  bool ok = true;

  if (warp < 8 && work) {
    // ---- softmax: thread = key tid % 128 of the tile, columns c0 .. c0 + C - 1 ----
    const int half = warp >> 2, c0 = half * C, w4 = warp & 3, at = tid & 127;
    const uint32_t lanes = tmem + ((uint32_t)(32 * w4) << 16);
    // The half's four warps agree: what some warp says; bit 1, a wait gave up.
    int ballots = 0;
    auto agree = [&](int what) {
      const int mine = what | (ok ? 0 : 2);
      int4 *v = &sh.vote[half][ballots++ & 1];
      if (lane == 0) reinterpret_cast<int *>(v)[w4] = mine;
      named_sync(1 + half, 128);
      const int4 x = *v;
      return x.x | x.y | x.z | x.w;
    };
    for (bool more = true; more && ok;) {
      const int row0 = u.rb * N;
      constexpr int kT = 128 / C < D / 32 ? 128 / C : D / 32, kGroups = D / 32 / kT;
      if (at < C * kT) {  // queries: kT threads a row
        const int n = c0 + at / kT, r = row0 + n, first = (at % kT) * kGroups;
        const bool live = r < u.rows;
        const int row = live ? r / p.group : 0, head = u.kvh * p.group + (live ? r % p.group : 0);
        const __nv_bfloat16 *q = p.q + u.b * p.q_sb + (int64_t)row * p.q_sl + (int64_t)head * p.q_sh;
        uint4 x[kGroups][4];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < kGroups; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            x[i][k] = live ? *reinterpret_cast<const uint4 *>(q + 32 * (first + i) + 8 * k) : make_uint4(0, 0, 0, 0);
            for (uint32_t v : {x[i][k].x, x[i][k].y, x[i][k].z, x[i][k].w})
              top = max(top, max((v << 16) & 0x7fff0000u, v & 0x7fff0000u));
          }
#pragma unroll
        for (int o = 1; o < kT; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        // the row's largest element to 2^14 .. 2^15: exact but for elements 2^20 times smaller
        const int up = top == 0 ? 0 : min(14 + 127 - (int)(top >> 23), 103);
        const float mul = __uint_as_float((uint32_t)(127 + up) << 23);
#pragma unroll
        for (int i = 0; i < kGroups; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) {  // dims k, k + 4, .. k + 28 of the group, as the codes' pairs have them
            auto dim = [&](int d) {
              const uint4 w = x[i][d >> 3];
              const uint32_t v = (d & 7) < 2 ? w.x : (d & 7) < 4 ? w.y : (d & 7) < 6 ? w.z : w.w;
              return __uint_as_float(d & 1 ? v & 0xffff0000u : v << 16) * mul;
            };
            const uint4 v = make_uint4(pack_f16(dim(k), dim(k + 4)), pack_f16(dim(k + 8), dim(k + 12)),
                                       pack_f16(dim(k + 16), dim(k + 20)), pack_f16(dim(k + 24), dim(k + 28)));
            const int gr = first + i, chunk = 4 * (gr & 1) + k;
            *reinterpret_cast<uint4 *>(sh.q + (gr >> 1) * (N * 128) + n * 128 + ((chunk ^ (n & 7)) << 4)) = v;
          }
        if (at % kT == 0) {
          float *col = reinterpret_cast<float *>(&sh.column[n >> 1]);
          col[n & 1] = logit_factor(p.scale_log2, up);
          col[2 + (n & 1)] = 0.f;
          sh.limit[n] = live ? (int)min((int64_t)u.seen, (int64_t)u.start + row + 1) : u.seen;
          sh.out_at[n] = u.b * p.o_sb + (int64_t)row * p.o_sl + (int64_t)head * p.o_sh;
          sh.lse_at[n] = (int)(((int64_t)u.b * p.Lq + row) * p.H + head);
        }
      }
      fence_proxy_async();
      named_sync(1 + half, 128);
      if (lane == 0) mbar_arrive(&sh.q_ready);
      const int least = (int)min((int64_t)u.seen, (int64_t)u.start + row0 / p.group + 1);
      uint64_t l[C / 2];
#pragma unroll
      for (int i = 0; i < C / 2; ++i) l[i] = 0;
      bool fresh = true, far = false;  // the references are still zero; as is_far has it
      for (int step = u.g0; step < u.g1; ++step, ++c) {
        const int st = c % ST, key = step * kTile + at;
        float f = 0.f, e = 0.f, w = 0.f;  // the key's factor of S, row exponent, 2^(kSumLift - e) or 0
        bool there = false, gone = false;
        if ((ok = mbar_wait_warp(&sh.full[st], (c / ST) & 1, abort))) {
          const uint32_t gran = smem_u32(sh.stage[st]) + (at >> 4) * G::kBytes;
          const int token = at & 15;
          uint32_t top = 0;
#pragma unroll
          for (int i = 0; i < J; ++i) {
            const uint2 s = lds64(gran + G::kKScales + token * (D / 16) + 8 * i);
            top = max(max(top, max(s.x << 16, s.x & 0xffff0000u)), max(s.y << 16, s.y & 0xffff0000u));
          }
          const uint32_t bits = lds16(gran + G::kVExps + 2 * token);
          const int missing = sh.gone[st];
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.empty[st]);
          f = __uint_as_float((uint32_t)(max((int)(top >> 23) & 255, 40) - 36) << 23);  // 2^E 2^-24
          gone = missing;
          there = key < u.seen && !((missing >> (at >> 4)) & 1);
          e = there ? __uint_as_float(bits << 16) : 0.f;
          w = there ? ex2(kSumLift - e) : 0.f;
        }
        const bool edge = step * kTile + kTile > least || gone;
        const uint32_t s_at = lanes + S::kS + (c & 1) * N + c0;
        ok = ok && mbar_wait_warp(&sh.s_full[c & 1], (c >> 1) & 1, abort);
        tc_fence_after();
        float y[C];  // logits less the columns' references
        bool up = false;
        if (ok) {
          tmem_load(s_at, y);
          tmem_wait_ld();
          const uint64_t f2 = pk2(f, f), e2 = pk2(e, e);
#pragma unroll
          for (int i = 0; i < C / 2; ++i) {
            const float4 col = sh.column[c0 / 2 + i];
            const uint64_t s2 = fmul2(pk2(y[2 * i], y[2 * i + 1]), f2);
            up2(ffma2(s2, pk2(col.x, col.y), fadd2(e2, pk2(col.z, col.w))), y[2 * i], y[2 * i + 1]);
          }
          if (edge) {
#pragma unroll
            for (int n = 0; n < C; ++n)
              if (!there || key >= sh.limit[c0 + n]) y[n] = -INFINITY;
          }
          float top = y[0];
#pragma unroll
          for (int n = 1; n + 1 < C; n += 2) top = fmax3(top, y[n], y[n + 1]);
          up = fmaxf(top, y[C - 1]) > (fresh ? kLowest : kLift4 + kRaise4);
          // P^T's buffer: the product that read it last is complete
          if (c >= 2) ok = mbar_wait_warp(&sh.pv_done[c & 1], ((c - 2) >> 1) & 1, abort);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.s_free[c & 1]);
        }
        int all = agree(__any_sync(0xffffffffu, up) || far ? 1 : 0);
        if (!(all & 2) && all) {
          // Move the references to kLift below the tile's largest logits: the first time there, later up only. A column that sees
          // no key of the first tile that has one sees none of the later ones either, and its reference counts for nothing.
          {
            float x[C];
#pragma unroll
            for (int n = 0; n < C; ++n) x[n] = fmaxf(y[n], kLowest);  // NaN counts as nothing
            const float most = fold(x, lane, [](float a, float b) { return fmaxf(a, b); });
            if (lane < C) sh.red[w4][c0 + lane] = most;
          }
          if (step > u.g0) ok = mbar_wait_warp(&sh.pv_done[(c - 1) & 1], ((c - 1) >> 1) & 1, abort);
          tc_fence_after();
          all = agree(__any_sync(0xffffffffu, is_far(w) && w > 0.f) ? 4 : 0);
          far = far || (all & 4);
          if (at < C) {
            const int n = c0 + at;
            const float most = fmaxf(fmaxf(sh.red[0][n], sh.red[1][n]), fmaxf(sh.red[2][n], sh.red[3][n]));
            const float by = most == kLowest ? 0.f : fresh ? most - kLift4 : fmaxf(most - kLift4, 0.f);
            reinterpret_cast<float *>(&sh.column[n >> 1])[2 + (n & 1)] -= by;
            sh.by[n] = by;
            sh.keep[n] = fresh ? 0.f : ex2(-0.5f * by);
          }
          named_sync(1 + half, 128);
          if (!(all & 2)) {
#pragma unroll
            for (int i = 0; i < C / 2; ++i) {
              const uint64_t half = *reinterpret_cast<const uint64_t *>(&sh.keep[c0 + 2 * i]);
              l[i] = fmul2(fmul2(l[i], half), half);  // their product may lie below 2^-126 and this above
              y[2 * i] -= sh.by[c0 + 2 * i];
              y[2 * i + 1] -= sh.by[c0 + 2 * i + 1];
            }
            if (step > u.g0 && !fresh) {
#pragma unroll 1
              for (int i = 0; i < J * C; i += 8) {
                const int n = i % C;
                const uint32_t o_at = lanes + S::kO + i / C * N + c0 + n;
                float o[8];
                tmem_ld8(o_at, o);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 8; ++k) o[k] *= sh.keep[c0 + n + k] * sh.keep[c0 + n + k];
                tmem_st8(o_at, o);
              }
              tmem_wait_st();
            }
            fresh = false;
            if (far) {  // the weights' own exponentials, and none left to w
              const float log_w = log2_of(w);
#pragma unroll
              for (int i = 0; i < C / 2; ++i) l[i] = fadd2(l[i], pk2(ex2(y[2 * i] + log_w), ex2(y[2 * i + 1] + log_w)));
              w = 0.f;
            }
          }
          tc_fence_before();
        }
        if (all & 2) {
          ok = false;
          break;
        }
        const uint64_t w2 = pk2(w, w);
        uint8_t *row = sh.pr[c & 1] + at * 128;
#pragma unroll
        for (int i = 0; i < C / 8; ++i) {
          uint32_t h[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float a = ex2(y[8 * i + 2 * k]), b = ex2(y[8 * i + 2 * k + 1]);
            l[4 * i + k] = ffma2(pk2(a, b), w2, l[4 * i + k]);
            h[k] = pack_f16(a, b);
          }
          *reinterpret_cast<uint4 *>(row + (((c0 / 8 + i) ^ (at & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.p_ready[c & 1]);
      }
      if (!ok) break;
      {  // the part's sums over the keys: lane n of a warp gets column n's
        float x[C];
#pragma unroll
        for (int i = 0; i < C / 2; ++i) up2(l[i], x[2 * i], x[2 * i + 1]);
        const float sum = fold(x, lane, [](float a, float b) { return a + b; });
        if (lane < C) sh.red[w4][c0 + lane] = sum;
      }
      ok = mbar_wait_warp(&sh.pv_done[(c - 1) & 1], ((c - 1) >> 1) & 1, abort) &&
           mbar_wait_warp(&sh.spoilt_ready[parts & 3], (parts >> 2) & 1, abort);
      tc_fence_after();
      if (agree(0) & 2) {
        ok = false;
        break;
      }
      const bool whole = u.g0 == 0 && u.g1 == u.n_steps;
      const int64_t slot = blockIdx.x + (int64_t)u.item * p.Hkv + u.kvh;
      const int cols = min(C, u.rows - row0 - c0);  // may be none
      if (at < cols) {
        const int n = c0 + at;
        const float sum = (sh.red[0][n] + sh.red[1][n]) + (sh.red[2][n] + sh.red[3][n]);
        const float m = sum == 0.f ? kLowest : -(reinterpret_cast<const float *>(&sh.column[n >> 1])[2 + (n & 1)]);
        sh.sum[n] = inverse_sum(sum);
        if (!whole)
          *reinterpret_cast<float2 *>(&p.part_ml[2 * (slot * N + n)]) = make_float2(m, sum);
        else if (p.lse)
          p.lse[sh.lse_at[n]] = log_sum(m, sum);
      }
      named_sync(1 + half, 128);
      // dims as the value codes' fragments have them: four neighbouring ones over two tiles of 16 lanes
      const int dim = 32 * w4 + 4 * (lane & 7) + 2 * (lane >> 4) + ((lane >> 3) & 1);
#pragma unroll 1
      for (int i = 0; i < J * C; i += 8) {
        const int n = i % C, d = dim + 128 * (i / C);
        if (n >= cols) continue;
        float o[8];
        tmem_ld8(lanes + S::kO + i / C * N + c0 + n, o);
        tmem_wait_ld();
        const int4 first = sh.spoilt[parts & 3][i / C * 4 + w4];
        const int spoilt = min(min(first.x, first.y), min(first.z, first.w));
        if (spoilt != 0x7fffffff) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (sh.limit[c0 + n + k] > spoilt) o[k] = __uint_as_float(0x7fffffffu);
        }
        if (whole) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (n + k < cols) p.out[sh.out_at[c0 + n + k] + d] = __float2bfloat16_rn(o[k] * sh.sum[c0 + n + k]);
        } else {
          float *to = &p.part_o[(slot * N + c0 + n) * D + d];
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (n + k < cols) to[k * D] = o[k];
        }
      }
      tc_fence_before();
      named_sync(1 + half, 128);  // the next part's queries take this one's place
      ++parts;
      more = !p.whole && u.find(p);
    }
  } else if (warp < 12 && work) {
    // ---- keys: warp 8 + w expands rows 32 w .. of the tile ----
    const int w4 = warp & 3;
    const uint32_t lanes = tmem + ((uint32_t)(32 * w4) << 16);
    for (bool more = true; more && ok; more = !p.whole && u.find(p)) {
      if (lane < D / 32) reinterpret_cast<int *>(&sh.spoilt[parts & 3][lane])[w4] = 0x7fffffff;  // a word of each is this warp's
      for (int step = u.g0; step < u.g1; ++step, ++c) {
        const int st = c % ST;
        ok = mbar_wait_warp(&sh.full[st], (c / ST) & 1, abort);
        if (ok && c >= KB) ok = mbar_wait_warp(&sh.s_full[(c - KB) & 1], ((c - KB) >> 1) & 1, abort);
        if (!ok) break;
        tc_fence_after();
        const uint32_t stage = smem_u32(sh.stage[st]), k_at = lanes + S::kK + (KB == 2 ? (c & 1) * (D / 2) : 0);
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          const uint32_t gran = stage + (2 * w4 + h) * G::kBytes;
          uint2 sa[J], sb[J];
          uint32_t ta = 0, tb = 0;  // rows g, g + 8: largest scale's bits
#pragma unroll
          for (int i = 0; i < J; ++i) {
            sa[i] = lds64(gran + G::kKScales + g * (D / 16) + 8 * i);
            sb[i] = lds64(gran + G::kKScales + (g + 8) * (D / 16) + 8 * i);
            ta = max(max(ta, max(sa[i].x << 16, sa[i].x & 0xffff0000u)), max(sa[i].y << 16, sa[i].y & 0xffff0000u));
            tb = max(max(tb, max(sb[i].x << 16, sb[i].x & 0xffff0000u)), max(sb[i].y << 16, sb[i].y & 0xffff0000u));
          }
          const int fa = max((int)(ta >> 23) & 255, 40), fb = max((int)(tb >> 23) & 255, 40);
          const float ma = __uint_as_float((uint32_t)(266 - fa) << 23), mb = __uint_as_float((uint32_t)(266 - fb) << 23);
#pragma unroll
          for (int i = 0; i < J; ++i) {
            const uint4 ka = lds128(gran + g * (D / 2) + 64 * i + 16 * t), kb = lds128(gran + (g + 8) * (D / 2) + 64 * i + 16 * t);
            const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
            for (int jp = 0; jp < 2; ++jp) {
              uint32_t r[16];
#pragma unroll
              for (int jj = 0; jj < 2; ++jj) {
                const uint32_t xa = jp ? sa[i].y : sa[i].x, xb = jp ? sb[i].y : sb[i].x;
                const uint32_t s[2] = {half2_of(__uint_as_float(jj ? xa & 0xffff0000u : xa << 16) * ma),
                                       half2_of(__uint_as_float(jj ? xb & 0xffff0000u : xb << 16) * mb)};
                const uint32_t w2[2] = {wa[2 * jp + jj], wb[2 * jp + jj]};
                const uint32_t lo = 0x000f000fu, hi = 0x00f000f0u, k = 0x64006400u;  // fp16 1024 + n, 1024 + 16 n
                const uint32_t off = 0x64086408u, sixteenth = 0x2c002c00u, m72 = 0xd480d480u;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const uint32_t v = w2[e], v8 = v >> 8;
                  r[8 * jj + e] = hmul2u(hsub2u(and_or(v, lo, k), off), s[e]);
                  r[8 * jj + 2 + e] = hmul2u(hfma2u(and_or(v, hi, k), sixteenth, m72), s[e]);
                  r[8 * jj + 4 + e] = hmul2u(hsub2u(and_or(v8, lo, k), off), s[e]);
                  r[8 * jj + 6 + e] = hmul2u(hfma2u(and_or(v8, hi, k), sixteenth, m72), s[e]);
                }
              }
              tmem_st_16x128b_x8(k_at + ((uint32_t)(16 * h) << 16) + 64 * i + 32 * jp, r);
            }
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.k_ready[c & 1]);
        if (edge_tile(step, u.seen)) {  // lane: a key
          const int key = step * kTile + 32 * w4 + lane, gi = 2 * w4 + (lane >> 4), token = lane & 15;
          const bool there = key < u.seen && !((sh.gone[st] >> gi) & 1);
#pragma unroll 1
          for (int j = 0; j < D / 32; ++j) {
            const uint32_t scale = lds16(stage + gi * G::kBytes + G::kVScales + ((token >> 1) * (D / 32) + j) * 4 + (token & 1) * 2);
            if (there && (scale & 0x7c00u) == 0x7c00u) atomicMin(reinterpret_cast<int *>(&sh.spoilt[parts & 3][j]) + w4, key);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.empty[st]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.spoilt_ready[parts & 3]);
      ++parts;
    }
  } else if (warp < 16 && work) {
    // ---- values: warp 12 + j expands the dims of group j of each 128 ----
    const int j = warp & 3;
    const uint32_t lanes = tmem + ((uint32_t)(32 * j) << 16);
    const uint32_t sel = j & 1 ? 0x7632 : 0x5410;
    for (bool more = true; more && ok; more = !p.whole && u.find(p)) {
      for (int step = u.g0; step < u.g1; ++step, ++c) {
        const int st = c % ST;
        ok = mbar_wait_warp(&sh.full[st], (c / ST) & 1, abort);
        if (ok && c >= VB) ok = mbar_wait_warp(&sh.pv_done[(c - VB) & 1], ((c - VB) >> 1) & 1, abort);
        if (!ok) break;
        tc_fence_after();
        const uint32_t stage = smem_u32(sh.stage[st]), v_at = lanes + S::kV + (VB == 2 ? (c & 1) * (D / 2) : 0);
        const int gone = sh.gone[st];
        const bool edge = edge_tile(step, u.seen) || gone;
#pragma unroll 1
        for (int i = 0; i < J; ++i)
#pragma unroll 1
          for (int quad = 0; quad < 2; ++quad) {  // four granules
            uint32_t a0[16], a1[16];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int gi = 4 * quad + k;
              const uint32_t gran = stage + gi * G::kBytes, at = gran + G::kVCodes + v_chunk(2 * t, 0, g) + 1024 * i;
              const uint4 va = lds128(at), vb = lds128(at + 512);  // token pairs t and t + 4
              const uint32_t scales = gran + G::kVScales + (t * (D / 32) + 4 * i + j) * 4;
              uint32_t ra = lds32(scales), rb = lds32(scales + D / 2);
              if (edge) {  // tokens that are not there: their memory may hold anything; values that are no numbers: see spoilt
                const int have = (gone >> gi) & 1 ? 0 : u.seen - step * kTile - kGranule * gi;
                ra &= (2 * t < have ? 0xffffu : 0u) | (2 * t + 1 < have ? 0xffff0000u : 0u);
                rb &= (2 * t + 8 < have ? 0xffffu : 0u) | (2 * t + 9 < have ? 0xffff0000u : 0u);
                ra = numbers(ra);
                rb = numbers(rb);
              }
              const uint32_t u0 = j < 2 ? __byte_perm(va.x, va.z, sel) : __byte_perm(va.y, va.w, sel);
              const uint32_t u1 = j < 2 ? __byte_perm(vb.x, vb.z, sel) : __byte_perm(vb.y, vb.w, sel);
              const uint32_t lo = 0x000f000fu, hi = 0x00f000f0u, one = 0x64006400u;
              const uint32_t off = 0x64086408u, sixteenth = 0x2c002c00u, m72 = 0xd480d480u;
              a0[4 * k] = hmul2u(hsub2u(and_or(u0, lo, one), off), ra);
              a0[4 * k + 1] = hmul2u(hfma2u(and_or(u0, hi, one), sixteenth, m72), ra);
              a0[4 * k + 2] = hmul2u(hsub2u(and_or(u1, lo, one), off), rb);
              a0[4 * k + 3] = hmul2u(hfma2u(and_or(u1, hi, one), sixteenth, m72), rb);
              a1[4 * k] = hmul2u(hsub2u(and_or(u0 >> 8, lo, one), off), ra);
              a1[4 * k + 1] = hmul2u(hfma2u(and_or(u0 >> 8, hi, one), sixteenth, m72), ra);
              a1[4 * k + 2] = hmul2u(hsub2u(and_or(u1 >> 8, lo, one), off), rb);
              a1[4 * k + 3] = hmul2u(hfma2u(and_or(u1 >> 8, hi, one), sixteenth, m72), rb);
            }
            tmem_st_16x128b_x8(v_at + 64 * i + 32 * quad, a0);
            tmem_st_16x128b_x8(v_at + (16u << 16) + 64 * i + 32 * quad, a1);
          }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&sh.v_ready[c & 1]);
          mbar_arrive(&sh.empty[st]);
        }
      }
    }
  } else if (warp == 16 && work) {
    // ---- copies: a lane a granule, page numbers four tiles ahead ----
    for (bool more = true; more && ok; more = !p.whole && u.find(p)) {
      int page = 0, granule = 0;
      bool wanted = false, there = false;
      for (int step = u.g0; step < u.g1; ++step, ++c) {
        const int slot = (step - u.g0) & 3, st = c % ST;
        if (slot == 0) {
          granule = kGs * step + lane;
          wanted = granule <= (u.seen - 1) / kGranule && granule < kGs * u.g1;
          if (wanted) {
            page = p.pv.table[(int64_t)u.b * p.pv.table_stride + (granule >> p.pv.page_shift)];
            there = (unsigned)page < (unsigned)p.pv.pages;
            if (!there) p.pv.fail();
          }
        }
        if (c >= ST && !(ok = mbar_wait_warp(&sh.empty[st], ((c / ST) - 1) & 1, abort))) break;
        const bool mine = wanted && (lane >> 3) == slot;
        const uint32_t copies = __ballot_sync(0xffffffffu, mine), missing = __ballot_sync(0xffffffffu, mine && !there);
        if (lane == 0) {
          sh.gone[st] = (int)(missing >> (8 * slot));
          mbar_expect_tx(&sh.full[st], __popc(copies) * G::kBytes);
        }
        __syncwarp();
        if (mine)  // a missing page: any bytes, none of which count
          bulk_load(sh.stage[st] + (lane & 7) * G::kBytes,
                    p.pv.pool + (int64_t)u.kvh * p.pv.head_bytes + (int64_t)(there ? page : 0) * p.pv.page_bytes +
                        (granule & ((1 << p.pv.page_shift) - 1)) * G::kBytes,
                    G::kBytes, &sh.full[st]);
      }
    }
  } else if (warp == 17 && work) {
    // ---- S^T = K Q^T ----
    const uint64_t desc = smem_desc_sw128(smem_u32(sh.q), 16, 1024);
    for (bool more = true; more && ok; more = !p.whole && u.find(p)) {
      ok = mbar_wait_warp(&sh.q_ready, parts++ & 1, abort);
      for (int step = u.g0; step < u.g1 && ok; ++step, ++c) {
        if (c >= 2 && !(ok = mbar_wait_warp(&sh.s_free[c & 1], ((c - 2) >> 1) & 1, abort))) break;
        if (!(ok = mbar_wait_warp(&sh.k_ready[c & 1], (c >> 1) & 1, abort))) break;
        tc_fence_after();
        if (lane == 0) {
          const uint32_t s_at = tmem + S::kS + (c & 1) * N, k_at = tmem + S::kK + (KB == 2 ? (c & 1) * (D / 2) : 0);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            mma_ts(s_at, k_at + 8 * kk, desc_join(desc_lo(desc) + (kk >> 2) * (N * 128 / 16) + (kk & 3) * 2, desc_hi(desc)),
                   idesc_f16(N, false), kk > 0);
          tc_commit(&sh.s_full[c & 1]);
        }
        __syncwarp();
      }
    }
  } else if (warp == 18 && work) {
    // ---- O^T += V^T P^T ---- (a thread of its own: one issues a product every 150 cycles, the tensor core takes 63)
    const uint64_t desc = smem_desc_sw128(smem_u32(sh.pr), 16, 1024);
    for (bool more = true; more && ok; more = !p.whole && u.find(p)) {
      for (int step = u.g0; step < u.g1; ++step, ++c) {
        ok = mbar_wait_warp(&sh.v_ready[c & 1], (c >> 1) & 1, abort) && mbar_wait_warp(&sh.p_ready[c & 1], (c >> 1) & 1, abort);
        if (!ok) break;
        tc_fence_after();
        if (lane == 0) {
          const uint32_t lo = desc_lo(desc) + (c & 1) * (kTile * 128 / 16);
          const uint32_t v_at = tmem + S::kV + (VB == 2 ? (c & 1) * (D / 2) : 0), add = step > u.g0;
#pragma unroll
          for (int i = 0; i < J; ++i)
#pragma unroll
            for (int kk = 0; kk < kTile / 16; ++kk)
              mma_ts(tmem + S::kO + i * N, v_at + 64 * i + 8 * kk, desc_join(lo + kk * 128, desc_hi(desc)), idesc_f16(N, true),
                     kk > 0 ? 1u : add);
          tc_commit(&sh.pv_done[c & 1]);
        }
        __syncwarp();
      }
    }
  }
  if ((warp == 17 || warp == 18) && !ok) {  // products under way end before TMEM is given back, or this long later
    if (lane == 0) tc_commit(&sh.drain[warp - 17]);
    const long long from = clock64();
    while (!mbar_test(&sh.drain[warp - 17], 0) && clock64() - from < kWaitCycles / 8) {
    }
    __syncwarp();
  }
  if (warp == 16 && !ok) {  // so do copies: the memory they write is this CTA's until then
    for (int i = max(0, c - ST); i < c; ++i) {
      const long long from = clock64();
      while (!mbar_test(&sh.full[i % ST], (i / ST) & 1) && clock64() - from < kWaitCycles / 8) {
      }
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && sh.abort && p.error) atomicMax(p.error, FPX_DEVICE_WAIT);
  if (warp == 16) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int D, int N>
int launch(PagedDecodeParams &p, const DecodeLayout &w, cudaStream_t stream) {
  constexpr int smem = sizeof(TcSmem<D, N>) + 1024;
  static_assert(smem <= 227 * 1024, "shared memory of one CTA");
  static std::atomic<uint64_t> set{0};
  return launch_decode<D, N / 8, kGs>(paged_decode_tc_kernel<D, N>, set, kTcThreads, smem, 1, p, w, stream);
}

}  // namespace

int launch_paged_decode_tc(PagedDecodeParams &p, const DecodeLayout &w, int d, cudaStream_t stream) {
  if (d == 256) return w.rows == 32 ? launch<256, 32>(p, w, stream) : launch<256, 64>(p, w, stream);
  return w.rows == 32 ? launch<128, 32>(p, w, stream) : launch<128, 64>(p, w, stream);
}

}  // namespace fpx
