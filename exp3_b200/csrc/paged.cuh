// Pages of the KV cache: byte layout of their two forms, shared by the kernels that write
// (paged_cache.cu) and read (paged_cache.cu, paged_decode.cu) them.
//
// The bytes of one page and KV head are granules of 16 tokens, each a multiple of 16 bytes, so
// one untiled bulk copy moves a granule's keys, values and scales into shared memory.
//
// bf16: 16 rows of [K d | V d]; the 16-byte chunk c of row t lies at place c ^ (t & 7) of its
// half, so ldmatrix reads eight rows without a bank conflict.
//
// int4, in this order:
//   K codes   16 x d/2 bytes. Row t: for each 128 dims, word (group j, part p) of 8 codes
//             (dims 32 j + 8 p .. + 7, low nibble first) lies at word 4 p + j: lane p of a quad
//             reads its parts of all four groups as 16 bytes, and a warp's eight rows are 512
//             contiguous bytes.
//   V codes   for each 128 dims: token pair q (8) x 128 bytes; the chunk of dims 32 j + 4 g .. + 3
//             (j = 0 .. 3) of both tokens lies at 16-byte place g ^ (2 (q & 3)): 8 bytes of the
//             even token, 8 of the odd one. The lanes (g, q) of a warp read without a conflict.
//   K scales  [16][d / 32] bf16; value = (code - 8) s, s = bf16(amax / 7).
//   V scales  [8 pairs][d / 32][2] fp16 and
//   V exps    [16] bf16 integers; value = (code - 8) r 2^e, e = floor(log2(row amax / 7)) in
//             [-60, 126], r = fp16(amax / 7 * 2^-e). r is below 2 whatever the values' size, so
//             the attention kernel multiplies it into fp16 probabilities; 2^e joins the logit.
// code = round-half-even(x / s) + 8, in 1 .. 15. A group with an infinity or a NaN reads back
// as NaN. The other groups of such a value row have the scales of exponent 126, which is zero below 2^101; where all are, the row's
// exponent is -60.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace fpx {

constexpr int kGranule = 16;  // tokens
constexpr int kSms = 148;

template <int FMT, int D>
struct Granule;
template <int D>
struct Granule<FPX_PAGES_BF16, D> {
  static constexpr int kRow = 4 * D;  // bytes of one token
  static constexpr int kBytes = kGranule * kRow;
};
template <int D>
struct Granule<FPX_PAGES_INT4, D> {
  static constexpr int kVCodes = kGranule * D / 2, kKScales = kGranule * D, kVScales = kKScales + D,
                       kVExps = kVScales + D, kBytes = kVExps + 2 * kGranule;
  static constexpr int kRow = kBytes / kGranule;
};

// Byte offset in the V codes of the 8 bytes of token t (in the granule), dims 128 J + 32 j + 4 g.
FPX_INLINE int v_chunk(int t, int J, int g) {
  const int q = t >> 1;
  return J * 1024 + q * 128 + ((g ^ (2 * (q & 3))) << 4) + ((t & 1) << 3);
}

// What the host checked about a pool and its page table.
struct PageView {
  uint8_t *pool;
  int64_t page_bytes, head_bytes;  // of one page; of one page and head
  int pages;                       // in the pool
  int page_shift;                  // log2(granules in a page)
  const int32_t *table;            // [B][max_pages]
  int64_t table_stride;
  int max_pages;
  const int32_t *starts, *counts;  // [B]; counts may be null: every row counts
  int *bad_index;                  // set where one of these names nothing; apart from the word of waits that gave up, whose
                                   // value other kernels take as a reason not to run. Null: not reported

  // Positions that the table holds; a tile's end stays below 2^31.
  FPX_INLINE int capacity() const { return (int)min((int64_t)max_pages << (page_shift + 4), (int64_t)0x7fffff80); }
  // Rows of sequence b that are no padding.
  FPX_INLINE int count(int b, int L) const {
    if (starts[b] < 0) return 0;
    return counts ? max(0, min(counts[b], L)) : L;
  }
  // The same with the start, both words read at once; a row past int32 positions counts, and fails where it is used.
  FPX_INLINE void rows(int b, int L, int &start, int &count) const {
    const int c = counts ? counts[b] : L;
    start = starts[b];
    count = start < 0 ? 0 : max(0, min(c, L));
  }
  FPX_INLINE void fail() const {
    if (bad_index) *bad_index = FPX_DEVICE_BAD_INDEX;
  }
};

// Host: element strides of a [B, L, heads, d] tensor; those of one-entry dims, which multiply
// nothing, as zero.
struct RowStrides {
  int64_t b, l, h;
  RowStrides(int64_t sb, int64_t sl, int64_t sh, int B, int L, int heads)
      : b(B > 1 ? sb : 0), l(L > 1 ? sl : 0), h(heads > 1 ? sh : 0) {}
  bool multiples_of(int n) const { return b % n == 0 && l % n == 0 && h % n == 0; }
};

// Host: fills a PageView and checks what can be checked there; returns an fpx_status.
int make_page_view(PageView *view, int format, const void *pool, int pages, int page_size, const int32_t *table,
                   int64_t table_stride, int max_pages, const int32_t *starts, const int32_t *counts, int Hkv, int d);

}  // namespace fpx
