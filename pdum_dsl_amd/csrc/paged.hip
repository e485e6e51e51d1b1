// A paged cache's rows: appending keys and values with their positions' rotation on the way, and reading them back.
//
// Append. A row's (heads_q + 2 heads_kv) heads are cut into chunks of 8 features, one or four a thread, whose features are
// alike; a chunk's partner in the rotation (features f and f + rotated / 2) is read by its own thread too, from the cache
// line that the neighbours have brought. y = x cos -+ partner sin in fp32, each product and the sum rounded (no fma): the
// same two roundings for both of a pair, and what elementary fp32 operations give. Then one rounding to the type, or to 4
// bits: four neighbouring threads hold a scale's 32 features, so its maximum takes two exchanges.
//
// Bytes bound it, each input read and each output written once, and before them the chain of loads to a token's place
// (starts, lengths, page), which is why a thread asks for all of its chunks first. 8 x 1024 tokens, 32/8 heads of 128, inputs
// in turn: 44.5 us, 202 MB (4.5 TB/s; 34 where they are in the last-level cache), with 1 / 2 / 3 / 6 chunks a thread 50 / 48 /
// 44 / 47; to 4 bits 35 there, 181 MB, with one chunk 41. Short calls have too few threads so: 64 single tokens 3.3 us with
// one, 4.0 with four (a launch).
#include "paged.h"

namespace pdh {
namespace {

constexpr int64_t kManyItems = 1024 * 256;  // us with one / four a thread: 49000 3.3 / 4.0, 110000 6.3 / 6.9, 390000 5.4 / 4.9

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

template <typename T, int D, int BITS, int NC>
__global__ __launch_bounds__(256) void paged_append(AppendArgs a) {
  constexpr int CPH = D / 8;  // chunks a head
  const int row = blockIdx.x;
  const int item0 = blockIdx.y * (256 * NC) + threadIdx.x;  // q's heads, then k's, then v's
  const int hkv = static_cast<int>(a.c.heads);
  const int heads = a.heads_q + 2 * hkv, half = a.rotated >> 1;
  const int f0 = item0 % CPH * 8;  // alike for all chunks of a thread
  const bool upper = f0 >= half;   // of a pair of halves
  auto head_of = [&](int j) { return (item0 + 256 * j) / CPH; };  // alike for four neighbours
  auto turned = [&](int head) { return head < a.heads_q + hkv && a.rotary && f0 < a.rotated; };
  u32x4 x[NC], px[NC];
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int head = head_of(j);
    x[j] = px[j] = u32x4{0u, 0u, 0u, 0u};
    if (head >= heads) continue;
    const uint16_t* src = head < a.heads_q         ? a.q + row * a.q_st + head * a.q_sh
                          : head < a.heads_q + hkv ? a.k + row * a.k_st + (head - a.heads_q) * a.k_sh
                                                   : a.v + row * a.v_st + (head - a.heads_q - hkv) * a.v_sh;
    x[j] = *reinterpret_cast<const u32x4*>(src + f0);
    if (turned(head) && !a.interleaved) px[j] = *reinterpret_cast<const u32x4*>(src + (upper ? f0 - half : f0 + half));
  }

  const int seq = seq_of_row(a.b, row);
  int pos = -1, page = -1;
  bool owned = false;
  if (seq < a.b.seqs) {
    const Seq s = seq_at(a.b, seq);
    owned = row >= s.row0 && row < s.row0 + s.n;
    pos = s.len - s.n + (row - s.row0);
    if (owned && (!a.rotary || pos < a.positions)) page = page_of(a.b, a.c, a.shift, seq, pos);
  }
  if (!owned && !a.zero_rest) return;
  if (owned && page < 0 && item0 == 0 && a.bad) atomicAdd(a.bad, 1);
  const bool nowhere = page < 0;  // of no sequence, or a token without a place
  const int in_page = pos & ((1 << a.shift) - 1);
  const int64_t place = nowhere ? 0 : pool_at<BITS>(a.c, page, in_page);
  const float* cs = a.rotary + pos * a.ld_rotary;
  f32x4u c[2], sn[2];  // of this thread's features: pairs (four of each), or halves (eight)
  if (!nowhere && a.rotary && f0 < a.rotated) {
    const int at = a.interleaved ? f0 >> 1 : (upper ? f0 - half : f0);
    c[0] = *reinterpret_cast<const f32x4u*>(cs + at);
    sn[0] = *reinterpret_cast<const f32x4u*>(cs + half + at);
    if (!a.interleaved) {
      c[1] = *reinterpret_cast<const f32x4u*>(cs + at + 4);
      sn[1] = *reinterpret_cast<const f32x4u*>(cs + half + at + 4);
    }
  }
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int head = head_of(j);
    if (head >= heads) break;
    const int kind = head < a.heads_q ? 0 : (head < a.heads_q + hkv ? 1 : 2);
    if (nowhere) {
      if (kind == 0) *reinterpret_cast<u32x4*>(a.qo + row * a.qo_st + head * a.qo_sh + f0) = u32x4{0u, 0u, 0u, 0u};
      continue;
    }
    u32x4 out = x[j];
    float y[8];
    unpack8<T>(x[j], y);
    if (turned(head)) {
#pragma clang fp contract(off)
      if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float u = y[2 * i], w = y[2 * i + 1];
          y[2 * i] = u * c[0][i] - w * sn[0][i];
          y[2 * i + 1] = w * c[0][i] + u * sn[0][i];
        }
      } else {
        float p[8];
        unpack8<T>(px[j], p);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float yc = y[i] * c[i >> 2][i & 3], ps = p[i] * sn[i >> 2][i & 3];
          y[i] = upper ? yc + ps : yc - ps;
        }
      }
      out = pack8<T>(y);
    }
    if (kind == 0) {
      *reinterpret_cast<u32x4*>(a.qo + row * a.qo_st + head * a.qo_sh + f0) = out;
      continue;
    }
    const int h = kind == 1 ? head - a.heads_q : head - a.heads_q - hkv;
    const int64_t at = place + h * a.c.sh;
    if constexpr (BITS == 16) {
      *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(kind == 1 ? a.c.k : a.c.v) + at + f0) = out;
    } else {
      uint32_t byte;
      const uint32_t codes = fp4_codes<T>(y, byte);
      *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(kind == 1 ? a.c.k : a.c.v) + at + f0 / 2) = codes;
      if ((f0 & 31) == 0) {
        const int64_t sp = scale_at(a.c, page, in_page) + h * a.c.ssh;
        static_cast<uint8_t*>(kind == 1 ? a.c.k_scale : a.c.v_scale)[sp + f0 / 32] = static_cast<uint8_t>(byte);
      }
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

// A chunk of 8 features a thread: 8 x 1024 tokens of 4 bits, 8 heads of 128, 12.5 us, 55 MB (4.4 TB/s); four, 13.9. 16 bits 13.4
// us, 67 MB that the last-level cache holds (5.0).
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

// f(chunks a thread): four where they fill the chip all the same, one where a call is short, or a row no more chunks than a
// workgroup has threads, which then take none but their first: 16/4 heads of 64, 192 chunks, us with one / four: 2000 rows
// 6.0 / 6.5, 8192 16.2 / 17.5, 16384 28.1 / 31.0 (4 bits 29.7 / 33.4); 12/12 heads of 64, 288 chunks: 1000 rows 5.5 / 4.9, 8192
// 26.6 / 19.4, 16384 48.5 / 34.0 (51.4 / 38.4).
template <typename F>
void by_chunks(int64_t rows, int64_t items, F f) {
  if (items > 256 && rows * items > kManyItems)
    f(std::integral_constant<int, 4>{});
  else
    f(std::integral_constant<int, 1>{});
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
  if (heads_q > 0) {  // chunks are read by other workgroups than write them, but where q_out is q
    const int64_t n = batch->rows, d = cache->features;
    const Tokens out{q_out, n, heads_q, d, qo_st, qo_sh}, in{q, n, heads_q, d, q_st, q_sh};
    const Spans o = out.spans();
    PDH_REQUIRE(o.apart(), PDH_EINVAL, "pdh_paged_append: q_out's rows overlap");
    PDH_REQUIRE((out.in_place_of(in) || o.apart_from(in.spans())) &&
                    o.apart_from(Tokens{k, n, cache->heads, d, k_st, k_sh}.spans()) &&
                    o.apart_from(Tokens{v, n, cache->heads, d, v_st, v_sh}.spans()),
                PDH_EINVAL, "pdh_paged_append: q_out overlaps k, v or q (it may be q, with q's strides)");
    PDH_REQUIRE(clear_of_cache(o, *cache), PDH_EINVAL, "pdh_paged_append: q_out overlaps the cache");
  }
  PDH_REQUIRE(pools_apart(*cache), PDH_EINVAL,
              "pdh_paged_append: rows of the cache's pools or scales overlap, or keys and values do");
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
  by_chunks(batch->rows, items, [&](auto nc) {
    constexpr int NC = decltype(nc)::value;
    const dim3 grid(static_cast<unsigned>(batch->rows), static_cast<unsigned>((items + 256 * NC - 1) / (256 * NC)));
    by_kind(*cache, [&](auto t, auto d, auto bits) {
      paged_append<decltype(t), decltype(d)::value, decltype(bits)::value, NC><<<grid, 256, 0, as_stream(stream)>>>(a);
    });
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
  const Spans ko = Tokens{k_out, batch->rows, cache->heads, cache->features, ko_st, ko_sh}.spans();
  const Spans vo = Tokens{v_out, batch->rows, cache->heads, cache->features, vo_st, vo_sh}.spans();
  PDH_REQUIRE(ko.apart() && vo.apart() && ko.apart_from(vo), PDH_EINVAL, "pdh_paged_rows: rows of the outputs overlap");
  PDH_REQUIRE(clear_of_cache(ko, *cache) && clear_of_cache(vo, *cache), PDH_EINVAL,
              "pdh_paged_rows: the outputs overlap the cache");
  const RowsArgs a{static_cast<uint16_t*>(k_out), static_cast<uint16_t*>(v_out), ko_st, ko_sh, vo_st, vo_sh, *cache,
                   *batch, shift, zero_rest != 0};
  const int64_t items = 2 * cache->heads * (cache->features / 8);
  const dim3 grid(static_cast<unsigned>(batch->rows), static_cast<unsigned>((items + 255) / 256));
  by_kind(*cache, [&](auto t, auto d, auto bits) {
    paged_rows<decltype(t), decltype(d)::value, decltype(bits)::value><<<grid, 256, 0, as_stream(stream)>>>(a);
  });
  return check_launch("pdh_paged_rows");
}
