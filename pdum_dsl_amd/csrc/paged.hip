// A paged cache's rows: appending keys and values with their positions' rotation on the way, and reading them back.
//
// Append. A row's (heads_q + 2 heads_kv) heads are cut into chunks of 8 features, one a thread; a chunk's partner in the
// rotation (features f and f + rotated / 2) is read by its own thread too, from the cache line that the neighbours have
// brought. y = x cos -+ partner sin in fp32, each product and the sum rounded (no fma): the same two roundings for both of a
// pair, and what elementary fp32 operations give. Then one rounding to the type, or to 4 bits: four neighbouring threads
// hold a scale's 32 features, so its maximum takes two exchanges. Bytes bound it: each input is read and each output
// written once. 8 x 1024 tokens, 32/8 heads of 128: 39 us, 202 MB (5.2 TB/s, as a copy of that size from memory); to 4 bits
// 41 us, 181 MB (4.4; VALU half busy with the rotation and the scales). 64 single tokens: 3.7 us, a launch. A workgroup
// takes chunks of one row, whose sequence is looked up once.
#include "paged.h"

namespace pdh {
namespace {

struct AppendArgs {
  const uint16_t *k, *v, *q;
  uint16_t* qo;
  int64_t k_st, k_sh, v_st, v_sh, q_st, q_sh, qo_st, qo_sh;
  pdh_paged_cache c;
  pdh_paged_batch b;
  const float* rotary;  // [positions][rotated]: cosines, then sines; NULL: nothing is rotated
  int64_t ld_rotary, positions;
  int rotated, interleaved, heads_q, shift, zero_rest;
  int* bad;
};

template <typename T>
__device__ __forceinline__ void unpack8(u32x4 x, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = lo_f32<T>(x[i]);
    f[2 * i + 1] = hi_f32<T>(x[i]);
  }
}

template <typename T>
__device__ __forceinline__ u32x4 pack8(const float (&f)[8]) {
  return u32x4{pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7])};
}

// Eight values of a 32-feature group that this thread shares with its three neighbours, as codes; the scale's byte is the
// least with max|y| <= 7 2^e, so that no rounding is off by more than half a step (7 lies half a step past 6), held to
// what the type of the cache's values can hold: 6 2^e <= 49152 in f16, 6 2^125 in bf16.
template <typename T>
__device__ __forceinline__ uint32_t fp4_codes(const float (&y)[8], uint32_t& byte) {
  uint32_t top = 0;  // the largest magnitude, as bits: infinities and NaN lie above every number
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t m = __float_as_uint(y[i]) & 0x7fffffffu;
    top = top > m ? top : m;
  }
#pragma unroll
  for (int off = 1; off <= 2; off <<= 1) {
    const uint32_t o = __shfl_xor(top, off, kWave);
    top = top > o ? top : o;
  }
  constexpr int kMost = (std::is_same_v<T, _Float16> ? 13 : 125) + 127;
  int e = static_cast<int>((top + 0x1fffffu) >> 23) - 2;  // the carry: a significand over 1.75
  e = e < 1 ? 1 : (e < kMost ? e : kMost);
  const bool finite = top < 0x7f800000u;
  byte = finite ? e : 255;
  // v_cvt_scalef32_pk_fp4_f32: two values over 2^(e - 127) to the nearest codes, ties to even ones, past 6 to 6
  const float scale = e8m0(e);
  uint32_t codes = 0;
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, y[0], y[1], scale, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, y[2], y[3], scale, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, y[4], y[5], scale, 2);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, y[6], y[7], scale, 3);
  return codes;
}

template <typename T, int D, int BITS>
__global__ __launch_bounds__(256) void paged_append(AppendArgs a) {
  constexpr int CPH = D / 8;  // chunks a head
  const int row = blockIdx.x;
  const int item = blockIdx.y * 256 + threadIdx.x;
  const int hkv = static_cast<int>(a.c.heads);
  const int head = item / CPH, f0 = item % CPH * 8;  // q's heads, then k's, then v's
  const bool live = head < a.heads_q + 2 * hkv;      // alike for four neighbours
  const int kind = head < a.heads_q ? 0 : (head < a.heads_q + hkv ? 1 : 2);
  const int h = kind == 0 ? head : (kind == 1 ? head - a.heads_q : head - a.heads_q - hkv);
  const uint16_t* src = kind == 0   ? a.q + row * a.q_st + h * a.q_sh
                        : kind == 1 ? a.k + row * a.k_st + h * a.k_sh
                                    : a.v + row * a.v_st + h * a.v_sh;
  const bool turn = kind < 2 && a.rotary && f0 < a.rotated;
  const int half = a.rotated >> 1;
  const bool upper = f0 >= half;  // of a pair of halves
  u32x4 x = {0u, 0u, 0u, 0u}, px = {0u, 0u, 0u, 0u};
  if (live) x = *reinterpret_cast<const u32x4*>(src + f0);
  if (live && turn && !a.interleaved) px = *reinterpret_cast<const u32x4*>(src + (upper ? f0 - half : f0 + half));

  const int seq = seq_of_row(a.b, row);
  if (!live) return;
  int pos = -1, page = -1;
  bool owned = false;
  if (seq < a.b.seqs) {
    const Seq s = seq_at(a.b, seq);
    owned = row >= s.row0 && row < s.row0 + s.n;
    pos = s.len - s.n + (row - s.row0);
    if (owned && (!a.rotary || pos < a.positions)) page = page_of(a.b, a.c, a.shift, seq, pos);
  }
  if (!owned && !a.zero_rest) return;
  if (owned && page < 0 && item == 0 && a.bad) atomicAdd(a.bad, 1);
  uint16_t* qo = a.qo + row * a.qo_st + h * a.qo_sh + f0;
  if (page < 0) {  // of no sequence, or a token without a place
    if (kind == 0) *reinterpret_cast<u32x4*>(qo) = u32x4{0u, 0u, 0u, 0u};
    return;
  }

  u32x4 out = x;
  float y[8];
  unpack8<T>(x, y);
  if (turn) {
#pragma clang fp contract(off)
    const float* cs = a.rotary + pos * a.ld_rotary;
    if (a.interleaved) {
      const f32x4u c = *reinterpret_cast<const f32x4u*>(cs + (f0 >> 1));
      const f32x4u s = *reinterpret_cast<const f32x4u*>(cs + half + (f0 >> 1));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float u = y[2 * i], w = y[2 * i + 1];
        y[2 * i] = u * c[i] - w * s[i];
        y[2 * i + 1] = w * c[i] + u * s[i];
      }
    } else {
      float p[8];
      unpack8<T>(px, p);
      const int at = upper ? f0 - half : f0;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const f32x4u c = *reinterpret_cast<const f32x4u*>(cs + at + 4 * j);
        const f32x4u s = *reinterpret_cast<const f32x4u*>(cs + half + at + 4 * j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float yc = y[4 * j + i] * c[i], ps = p[4 * j + i] * s[i];
          y[4 * j + i] = upper ? yc + ps : yc - ps;
        }
      }
    }
    out = pack8<T>(y);
  }
  if (kind == 0) {
    *reinterpret_cast<u32x4*>(qo) = out;
    return;
  }
  const int in_page = pos & ((1 << a.shift) - 1);
  const int64_t place = pool_at<BITS>(a.c, page, in_page) + h * a.c.sh;
  if constexpr (BITS == 16) {
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(kind == 1 ? a.c.k : a.c.v) + place + f0) = out;
  } else {
    uint32_t byte;
    const uint32_t codes = fp4_codes<T>(y, byte);
    *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(kind == 1 ? a.c.k : a.c.v) + place + f0 / 2) = codes;
    if ((f0 & 31) == 0) {
      const int64_t sp = scale_at(a.c, page, in_page) + h * a.c.ssh;
      static_cast<uint8_t*>(kind == 1 ? a.c.k_scale : a.c.v_scale)[sp + f0 / 32] = static_cast<uint8_t>(byte);
    }
  }
}

struct RowsArgs {
  uint16_t *ko, *vo;
  int64_t ko_st, ko_sh, vo_st, vo_sh;
  pdh_paged_cache c;
  pdh_paged_batch b;
  int shift, zero_rest;
};

// A chunk of 8 features a thread, as above: 8 x 1024 tokens of 4 bits 12.4 us, 55 MB (4.4 TB/s).
template <typename T, int D, int BITS>
__global__ __launch_bounds__(256) void paged_rows(RowsArgs a) {
  constexpr int CPH = D / 8;
  const int row = blockIdx.x;
  const int item = blockIdx.y * 256 + threadIdx.x;
  const int hkv = static_cast<int>(a.c.heads);
  const int head = item / CPH, f0 = item % CPH * 8;
  const bool isk = head < hkv;
  const int h = isk ? head : head - hkv;
  const int seq = seq_of_row(a.b, row);
  if (head >= 2 * hkv) return;
  int pos = -1, page = -1;
  bool owned = false;
  if (seq < a.b.seqs) {
    const Seq s = seq_at(a.b, seq);
    owned = row >= s.row0 && row < s.row0 + s.n;
    pos = s.len - s.n + (row - s.row0);
    if (owned) page = page_of(a.b, a.c, a.shift, seq, pos);
  }
  if (!owned && !a.zero_rest) return;
  u32x4 x = {0u, 0u, 0u, 0u};
  if (page >= 0) {
    const int in_page = pos & ((1 << a.shift) - 1);
    const int64_t place = pool_at<BITS>(a.c, page, in_page) + h * a.c.sh;
    if constexpr (BITS == 16) {
      x = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(isk ? a.c.k : a.c.v) + place + f0);
    } else {
      const int64_t sp = scale_at(a.c, page, in_page) + h * a.c.ssh;
      const uint32_t codes =
          *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(isk ? a.c.k : a.c.v) + place + f0 / 2);
      x = fp4_row8<T>(codes, e8m0(static_cast<const uint8_t*>(isk ? a.c.k_scale : a.c.v_scale)[sp + f0 / 32]));
    }
  }
  uint16_t* out = isk ? a.ko + row * a.ko_st + h * a.ko_sh : a.vo + row * a.vo_st + h * a.vo_sh;
  *reinterpret_cast<u32x4*>(out + f0) = x;
}

}  // namespace
}  // namespace pdh

using namespace pdh;

extern "C" int pdh_paged_append(const void* k, const void* v, const void* q, void* q_out, int64_t heads_q, int64_t k_st,
                                int64_t k_sh, int64_t v_st, int64_t v_sh, int64_t q_st, int64_t q_sh, int64_t qo_st,
                                int64_t qo_sh, const pdh_paged_cache* cache, const pdh_paged_batch* batch,
                                const float* rotary, int64_t positions, int64_t rotated, int64_t ld_rotary,
                                int interleaved, int zero_rest, int* bad, void* stream) {
  int shift = 0;
  const int rc = check_paged("pdh_paged_append", cache, batch, &shift);
  if (rc) return rc;
  PDH_REQUIRE(heads_q >= 0 && heads_q <= 65535, PDH_EINVAL, "pdh_paged_append: bad number of query heads");
  if (batch->rows == 0) return PDH_OK;
  PDH_REQUIRE((q == nullptr) == (heads_q == 0) && (q_out == nullptr) == (heads_q == 0), PDH_EINVAL,
              "pdh_paged_append: q and q_out come together, with heads_q >= 1");
  PDH_REQUIRE(k && v && aligned16(k) && aligned16(v) && aligned16(q) && aligned16(q_out), PDH_EINVAL,
              "pdh_paged_append: k, v, q and q_out must be 16-byte aligned");
  for (int64_t s : {k_st, k_sh, v_st, v_sh, q_st, q_sh, qo_st, qo_sh})
    PDH_REQUIRE(s >= 0 && s % 8 == 0, PDH_EINVAL, "pdh_paged_append: strides must be multiples of 8 elements, >= 0");
  if (rotary) {
    PDH_REQUIRE(rotated >= 16 && rotated % 16 == 0 && rotated <= cache->features, PDH_EUNSUPPORTED,
                "pdh_paged_append: rotated must be a multiple of 16 in [16, features] (got %lld)", (long long)rotated);
    PDH_REQUIRE(positions >= 0 && ld_rotary >= rotated, PDH_EINVAL, "pdh_paged_append: bad rotary table");
  }
  const AppendArgs a{static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), static_cast<const uint16_t*>(q),
                     static_cast<uint16_t*>(q_out), k_st, k_sh, v_st, v_sh, q_st, q_sh, qo_st, qo_sh, *cache, *batch,
                     rotary, ld_rotary, positions, static_cast<int>(rotary ? rotated : 0), interleaved != 0,
                     static_cast<int>(heads_q), shift, zero_rest != 0, bad};
  const int64_t items = (heads_q + 2 * cache->heads) * (cache->features / 8);
  const dim3 grid(static_cast<unsigned>(batch->rows), static_cast<unsigned>((items + 255) / 256));
  by_kind(*cache, [&](auto t, auto d, auto bits) {
    paged_append<decltype(t), decltype(d)::value, decltype(bits)::value><<<grid, 256, 0, as_stream(stream)>>>(a);
  });
  return check_launch("pdh_paged_append");
}

extern "C" int pdh_paged_rows(void* k_out, void* v_out, int64_t ko_st, int64_t ko_sh, int64_t vo_st, int64_t vo_sh,
                              const pdh_paged_cache* cache, const pdh_paged_batch* batch, int zero_rest, void* stream) {
  int shift = 0;
  const int rc = check_paged("pdh_paged_rows", cache, batch, &shift);
  if (rc) return rc;
  if (batch->rows == 0) return PDH_OK;
  PDH_REQUIRE(k_out && v_out && aligned16(k_out) && aligned16(v_out), PDH_EINVAL,
              "pdh_paged_rows: the outputs must be 16-byte aligned");
  for (int64_t s : {ko_st, ko_sh, vo_st, vo_sh})
    PDH_REQUIRE(s >= 0 && s % 8 == 0, PDH_EINVAL, "pdh_paged_rows: strides must be multiples of 8 elements, >= 0");
  const RowsArgs a{static_cast<uint16_t*>(k_out), static_cast<uint16_t*>(v_out), ko_st, ko_sh, vo_st, vo_sh, *cache,
                   *batch, shift, zero_rest != 0};
  const int64_t items = 2 * cache->heads * (cache->features / 8);
  const dim3 grid(static_cast<unsigned>(batch->rows), static_cast<unsigned>((items + 255) / 256));
  by_kind(*cache, [&](auto t, auto d, auto bits) {
    paged_rows<decltype(t), decltype(d)::value, decltype(bits)::value><<<grid, 256, 0, as_stream(stream)>>>(a);
  });
  return check_launch("pdh_paged_rows");
}
