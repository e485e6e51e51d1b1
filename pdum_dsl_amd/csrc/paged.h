// What the paged-cache kernels share: the cache's and the batch's descriptions, where a token lies, and the 4-bit rows.
//
// Cache: pools [pages][heads][page_rows][features]; token s of sequence i lies in page table[i][s / page_rows], row
// s % page_rows. Batch: sequence i's new tokens are rows starts[i] .. starts[i + 1] - 1 of the call's tensors and the last
// of its lengths[i] tokens. starts, lengths and the table are device memory that no host code has seen, so every kernel
// clamps what it derives from them: rows to [0, rows), keys to the table's reach, page numbers to the pool. A row's position
// goes by starts as it stands, lengths[i] - (starts[i + 1] - row), whether or not the rows behind it are there.
#pragma once

#include "common.h"
#include "spans.h"

#include <initializer_list>
#include <type_traits>

namespace pdh {

constexpr int kMaxTokens = 1 << 30;  // a table's reach: positions and keys are 32-bit
// Lengths count as no more: the positions of up to 2^24 rows that end there are all past every table, and a window from
// them, another 2^30 back, is still a 32-bit number.
constexpr int kMaxLength = kMaxTokens + (1 << 24);

// One sequence's part of a batch.
struct Seq {
  int row0, n;  // its first row and number of new tokens
  int len;      // tokens in the cache up to its last row that is there, in [0, kMaxLength]; 0 where all rows lie before it
};

__device__ __forceinline__ int clamp_row(int r, int rows) { return r < 0 ? 0 : (r < rows ? r : rows); }

__device__ __forceinline__ Seq seq_at(const pdh_paged_batch& b, int i) {
  const int rows = static_cast<int>(b.rows);
  const int end = b.starts[i + 1], r0 = clamp_row(b.starts[i], rows), r1 = clamp_row(end, rows);
  const int held = b.lengths[i];
  const int len = (held > 0 ? held : 0) - (end > rows ? end - rows : 0);  // less the tokens whose rows are not there
  return Seq{r0, r1 > r0 ? r1 - r0 : 0, len < 0 ? 0 : (len < kMaxLength ? len : kMaxLength)};
}

// The sequence that owns a row: the number of sequences that end at or before it (seqs: none owns it). One wave, every
// lane the same row; 64 sequences a load. Every wave of a call reads them all: an append of single tokens, 4/2 heads of 64, takes
// 3.1 / 5.1 / 32 / 419 us for 64 / 700 / 4096 / 16384 sequences.
__device__ __forceinline__ int seq_of_row(const pdh_paged_batch& b, int row) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int64_t i = 0; i < b.seqs; i += 64) {
    const bool before = i + lane < b.seqs && b.starts[i + lane + 1] <= row;
    n += __popcll(__builtin_amdgcn_ballot_w64(before));
  }
  return __builtin_amdgcn_readfirstlane(n);
}

// The page of token s of sequence i, or -1 where the table or the pool has none.
__device__ __forceinline__ int page_of(const pdh_paged_batch& b, const pdh_paged_cache& c, int shift, int i, int s) {
  const int at = s >> shift;
  if (s < 0 || at >= b.width) return -1;
  const int p = b.table[i * b.ld_table + at];
  return static_cast<uint32_t>(p) < static_cast<uint64_t>(c.pages) ? p : -1;
}

// Where a row of a page lies in either pool, from a head's first row: units of the pools (16-bit elements, bytes), and
// bytes of the scales. A page's distance is a 32-bit number of 16 bytes (the pools') or bytes (the scales').
template <int BITS>
__device__ __forceinline__ int64_t pool_at(const pdh_paged_cache& c, int page, int in_page) {
  constexpr int unit = BITS == 16 ? 8 : 16;
  return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(page)) * static_cast<uint32_t>(c.sp / unit)) * unit +
         in_page * static_cast<int>(c.sr);
}
__device__ __forceinline__ int64_t scale_at(const pdh_paged_cache& c, int page, int in_page) {
  return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(page)) * static_cast<uint32_t>(c.ssp)) +
         in_page * static_cast<int>(c.ssr);
}

// ---- 4 bits: e2m1 codes (sign, two bits of exponent, one of mantissa: 0 .5 1 1.5 2 3 4 6), two a byte, the even feature
// in the low half; 32 features share the scale 2^(byte - 127), byte 255: NaN. gfx950 converts pairs of them, scaled, in
// one instruction (byte 255 gives NaN for every code, byte 0 is 2^-127).

__device__ __forceinline__ float e8m0(uint32_t byte) { return __uint_as_float(byte << 23); }

template <typename T, int I>
__device__ __forceinline__ uint32_t fp4_pair(uint32_t codes, float scale) {
  if constexpr (std::is_same_v<T, _Float16>)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, I));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, I));
}

// Eight codes as eight 16-bit values.
template <typename T>
__device__ __forceinline__ u32x4 fp4_row8(uint32_t codes, float scale) {
  return u32x4{fp4_pair<T, 0>(codes, scale), fp4_pair<T, 1>(codes, scale), fp4_pair<T, 2>(codes, scale),
               fp4_pair<T, 3>(codes, scale)};
}

// ---- host

// The checks that every entry point makes of a cache and a batch; the page's log2.
inline int check_paged(const char* fn, const pdh_paged_cache* c, const pdh_paged_batch* b, int* shift) {
  PDH_REQUIRE(c && b, PDH_EINVAL, "%s: null cache or batch", fn);
  PDH_REQUIRE(c->dtype == PDH_BF16 || c->dtype == PDH_F16, PDH_EUNSUPPORTED, "%s: dtype must be bf16 or f16", fn);
  PDH_REQUIRE(c->bits == 16 || c->bits == 4, PDH_EUNSUPPORTED, "%s: a cache has 16 or 4 bits (got %d)", fn, c->bits);
  PDH_REQUIRE(c->features == 64 || c->features == 128, PDH_EUNSUPPORTED, "%s: features must be 64 or 128 (got %lld)", fn,
              (long long)c->features);
  PDH_REQUIRE(c->pages >= 1 && c->pages <= INT32_MAX && c->heads >= 1 && c->heads <= 65535, PDH_EINVAL,
              "%s: bad number of pages or heads", fn);
  const int64_t p = c->page_rows;
  PDH_REQUIRE(p >= 16 && p <= 4096 && (p & (p - 1)) == 0, PDH_EUNSUPPORTED,
              "%s: page_rows must be a power of two in [16, 4096] (got %lld)", fn, (long long)p);
  PDH_REQUIRE(c->k && c->v && aligned16(c->k) && aligned16(c->v), PDH_EINVAL, "%s: pools must be 16-byte aligned", fn);
  const int64_t unit = c->bits == 4 ? 16 : 8;  // 16 bytes
  const int64_t row = c->bits == 4 ? c->features / 2 : c->features;
  for (int64_t s : {c->sp, c->sh, c->sr})
    PDH_REQUIRE(s >= 0 && s % unit == 0, PDH_EINVAL, "%s: the pools' strides must be multiples of 16 bytes, >= 0", fn);
  PDH_REQUIRE(c->sr >= row && c->sr < (1 << 16), PDH_EINVAL, "%s: the pools' rows overlap or lie 2^16 or more apart", fn);
  PDH_REQUIRE(c->sp / unit < INT32_MAX && c->sh < INT64_MAX / 65536 / 2, PDH_EINVAL,
              "%s: the pools' pages lie 2^35 bytes or more apart", fn);
  if (c->bits == 4) {
    PDH_REQUIRE(c->k_scale && c->v_scale, PDH_EINVAL, "%s: a 4-bit cache needs its scales", fn);
    PDH_REQUIRE(c->ssp >= 0 && c->ssh >= 0 && c->ssp <= INT32_MAX, PDH_EINVAL,
                "%s: the scales' strides must be >= 0, pages less than 2^31 bytes apart", fn);
    PDH_REQUIRE(c->ssr >= c->features / 32 && c->ssr < (1 << 16), PDH_EINVAL,
                "%s: the scales' rows overlap or lie 2^16 or more apart", fn);
  }
  PDH_REQUIRE(b->seqs >= 0 && b->seqs <= (1 << 20) && b->rows >= 0 && b->rows < (1 << 24), PDH_EINVAL,
              "%s: at most 2^20 sequences and 2^24 - 1 rows", fn);
  PDH_REQUIRE(b->width >= 0 && b->width * p <= kMaxTokens && b->ld_table >= 0, PDH_EINVAL,
              "%s: a table reaches at most 2^30 tokens", fn);
  if (b->seqs > 0)
    PDH_REQUIRE((b->table || b->width == 0) && b->starts && b->lengths, PDH_EINVAL, "%s: null table, starts or lengths", fn);
  *shift = __builtin_ctzll(static_cast<unsigned long long>(p));
  return PDH_OK;
}

// Whether no two rows of a cache's pools, and of its scales, share a byte: an append stores several otherwise in one place,
// and which of them stays goes by the order of the workgroups. Keys and values are one array more, two entries long: they
// may lie in one tensor.
inline bool pools_apart(const pdh_paged_cache& c) {
  auto apart = [&](const void* k, const void* v, int64_t row, int64_t page, int64_t head, int64_t in_page) {
    const intptr_t between = reinterpret_cast<intptr_t>(v) - reinterpret_cast<intptr_t>(k);
    return Spans(k, row, {{c.pages, page}, {c.heads, head}, {c.page_rows, in_page}, {2, between < 0 ? -between : between}})
        .apart();
  };
  if (c.bits == 16) return apart(c.k, c.v, c.features * 2, c.sp * 2, c.sh * 2, c.sr * 2);
  return apart(c.k, c.v, c.features / 2, c.sp, c.sh, c.sr) &&
         apart(c.k_scale, c.v_scale, c.features / 32, c.ssp, c.ssh, c.ssr);
}

// Whether an output shares no byte with the cache's pools and scales, which other workgroups read.
inline bool clear_of_cache(const Spans& out, const pdh_paged_cache& c) {
  auto clear = [&](const void* p, int64_t row, int64_t page, int64_t head, int64_t in_page) {
    return out.apart_from(Spans(p, row, {{c.pages, page}, {c.heads, head}, {c.page_rows, in_page}}));
  };
  const int64_t es = c.bits == 16 ? 2 : 1, row = c.features * c.bits / 8;
  for (const void* p : {c.k, c.v})
    if (!clear(p, row, c.sp * es, c.sh * es, c.sr * es)) return false;
  if (c.bits == 4)
    for (const void* p : {c.k_scale, c.v_scale})
      if (!clear(p, c.features / 32, c.ssp, c.ssh, c.ssr)) return false;
  return true;
}

// A [rows][heads][features] tensor of 16-bit elements.
struct Tokens {
  const void* p;
  int64_t rows, heads, features, st, sh;
  Spans spans() const { return Spans(p, features * 2, {{rows, st * 2}, {heads, sh * 2}}); }
  bool in_place_of(const Tokens& o) const {  // of the same sizes
    return p == o.p && (rows <= 1 || st == o.st) && (heads <= 1 || sh == o.sh);
  }
};

// f(element type, features, bits) of a cache.
template <typename F>
void by_kind(const pdh_paged_cache& c, F f) {
  using std::integral_constant;
  auto bits = [&](auto t, auto d) {
    if (c.bits == 16)
      f(t, d, integral_constant<int, 16>{});
    else
      f(t, d, integral_constant<int, 4>{});
  };
  auto dim = [&](auto t) {
    if (c.features == 128)
      bits(t, integral_constant<int, 128>{});
    else
      bits(t, integral_constant<int, 64>{});
  };
  if (c.dtype == PDH_BF16)
    dim(__hip_bfloat16{});
  else
    dim(_Float16{});
}

}  // namespace pdh
