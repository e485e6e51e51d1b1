// Attention over a paged cache: rows of several sequences, causal, with an optional window and first tokens kept.
//
//   x(p, s) = scale q_p . k_s over the visible s: s <= p and (s < sinks or s > p - window)
//   o = sum_s softmax(x) v_s, lse = log sum_s exp x;  a row with no visible key: o = 0, lse = -inf
//
// Row kernel: a wave per (row, query head), keys 64 at a time, one a lane; the online softmax's maximum and sum are the
// wave's, o's features lie across its lanes. It touches no key that the row does not see.
#include "paged.h"

#include <cmath>
namespace pdh {
namespace {

constexpr float kInf = __builtin_inff();

struct PagedAttn {
  const uint16_t* q;
  uint16_t* o;
  float* lse;  // [rows][heads_q], may be NULL
  int64_t q_st, q_sh, o_st, o_sh;
  pdh_paged_cache c;
  pdh_paged_batch b;
  int heads_q, group;  // group: query heads a key/value head
  int window, sinks;
  int shift, zero_rest;
  int reach;  // keys that the table has pages for
  float c2;   // scale * log2(e)
};

// One row's softmax state over the visible keys of [k0, k1): m in units of log2, o unnormalised, features lane + 64 j.
template <typename T, int D, int BITS>
__device__ void row_sweep(const PagedAttn& a, int seq, int hk, const uint16_t* q, int pos, int k0, int k1, float& m,
                          float& l, float (&o)[D / 64]) {
  const int lane = threadIdx.x & 63;
  const int mask = (1 << a.shift) - 1;
  k1 = k1 < pos + 1 ? k1 : pos + 1;
  k1 = k1 < a.reach ? k1 : a.reach;
  for (int kb = k0; kb < k1; kb += kWave) {
    if (kb >= a.sinks && kb + kWave - 1 <= pos - a.window) {  // behind the first tokens, before the window
      const int next = pos - a.window + 1;
      kb = kb + (next - kb) / kWave * kWave;
      if (kb >= k1) break;
    }
    const int key = kb + lane;
    int page = -1;
    if (key < k1 && (key < a.sinks || key > pos - a.window)) page = page_of(a.b, a.c, a.shift, seq, key);
    const bool seen = page >= 0;
    const unsigned long long live = __builtin_amdgcn_ballot_w64(seen);
    if (live == 0) continue;
    const int64_t kat = seen ? page * a.c.k_sp + hk * a.c.k_sh + (key & mask) * a.c.k_sr : 0;
    const int64_t vat = seen ? page * a.c.v_sp + hk * a.c.v_sh + (key & mask) * a.c.v_sr : 0;
    const int64_t ksat = seen ? page * a.c.ks_sp + hk * a.c.ks_sh + (key & mask) * a.c.ks_sr : 0;
    const int64_t vsat = seen ? page * a.c.vs_sp + hk * a.c.vs_sh + (key & mask) * a.c.vs_sr : 0;
    float x = -kInf;
    if (seen) {
      float dot = 0.f;
#pragma unroll 2
      for (int f = 0; f < D; f += 8) {
        u32x4 kk;
        if constexpr (BITS == 16) {
          kk = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.c.k) + kat + f);
        } else {
          kk = fp4_row8<T>(*reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.c.k) + kat + f / 2),
                           e8m0(static_cast<const uint8_t*>(a.c.k_scale)[ksat + f / 32]));
        }
        const u32x4 qq = *reinterpret_cast<const u32x4*>(q + f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          dot = __builtin_fmaf(lo_f32<T>(qq[i]), lo_f32<T>(kk[i]), dot);
          dot = __builtin_fmaf(hi_f32<T>(qq[i]), hi_f32<T>(kk[i]), dot);
        }
      }
      x = dot * a.c2;
    }
    // a NaN score stays in x: its exponential is NaN, and so is the row
    const float mnew = fmaxf(m, wave_max(x));
    const float ref = mnew == -kInf ? 0.f : mnew;  // scores of -inf alone weigh 0, not NaN
    const float alpha = fast_exp2(m - ref);
    const float p = seen ? fast_exp2(x - ref) : 0.f;
    l = l * alpha + wave_sum(p);
    m = mnew;
#pragma unroll
    for (int j = 0; j < D / 64; ++j) o[j] *= alpha;
    for (unsigned long long todo = live; todo; todo &= todo - 1) {
      const int kk = __builtin_ctzll(todo);
      const float pk = __shfl(p, kk, kWave);
      const int64_t at = (static_cast<int64_t>(__shfl(static_cast<int>(vat >> 32), kk, kWave)) << 32) |
                         static_cast<uint32_t>(__shfl(static_cast<int>(vat), kk, kWave));
      if constexpr (BITS == 16) {
        const uint16_t* v = static_cast<const uint16_t*>(a.c.v) + at;
#pragma unroll
        for (int j = 0; j < D / 64; ++j) o[j] = __builtin_fmaf(pk, Elem<T>::to_f32(v[lane + 64 * j]), o[j]);
      } else {
        const int64_t sat = (static_cast<int64_t>(__shfl(static_cast<int>(vsat >> 32), kk, kWave)) << 32) |
                            static_cast<uint32_t>(__shfl(static_cast<int>(vsat), kk, kWave));
        const uint8_t* v = static_cast<const uint8_t*>(a.c.v) + at;
        const uint8_t* sc = static_cast<const uint8_t*>(a.c.v_scale) + sat;
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
          const int f = lane + 64 * j;
          const uint32_t code = v[f >> 1] >> (4 * (f & 1));
          o[j] = __builtin_fmaf(pk, lo_f32<T>(fp4_pair<T, 0>(code, e8m0(sc[f / 32]))), o[j]);
        }
      }
    }
  }
}

template <typename T, int D, int BITS>
__global__ __launch_bounds__(256) void paged_attn_rows(PagedAttn a) {
  const int lane = threadIdx.x & 63;
  const int row = blockIdx.x;
  const int h = blockIdx.y * 4 + wave_id();
  if (h >= a.heads_q) return;
  const int seq = seq_of_row(a.b, row);
  Seq s{0, 0, 0};
  bool owned = false;
  if (seq < a.b.seqs) {
    s = seq_at(a.b, seq);
    owned = row >= s.row0 && row < s.row0 + s.n;
  }
  if (!owned && !a.zero_rest) return;
  float m = -kInf, l = 0.f, o[D / 64] = {};
  if (owned)
    row_sweep<T, D, BITS>(a, seq, h / a.group, a.q + row * a.q_st + h * a.q_sh, s.len - s.n + (row - s.row0), 0,
                          kMaxTokens, m, l, o);
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  uint16_t* out = a.o + row * a.o_st + h * a.o_sh;
#pragma unroll
  for (int j = 0; j < D / 64; ++j) out[lane + 64 * j] = Elem<T>::from_f32(o[j] * inv);
  if (lane == 0 && a.lse) a.lse[static_cast<int64_t>(row) * a.heads_q + h] = l == 0.f ? -kInf : (m + __log2f(l)) * kLn2;
}

}  // namespace
}  // namespace pdh

using namespace pdh;

extern "C" size_t pdh_paged_attention_workspace(const pdh_paged_cache* cache, const pdh_paged_batch* batch,
                                                int64_t heads_q, int64_t window, int64_t sinks) {
  (void)cache, (void)batch, (void)heads_q, (void)window, (void)sinks;
  return 0;
}

extern "C" int pdh_paged_attention(const void* q, void* o, float* lse, int64_t heads_q, int64_t q_st, int64_t q_sh,
                                   int64_t o_st, int64_t o_sh, const pdh_paged_cache* cache,
                                   const pdh_paged_batch* batch, int64_t window, int64_t sinks, float scale,
                                   int zero_rest, void* ws, size_t ws_bytes, void* stream) {
  (void)ws, (void)ws_bytes;
  int shift = 0;
  const int rc = check_paged("pdh_paged_attention", cache, batch, &shift);
  if (rc) return rc;
  PDH_REQUIRE(heads_q >= 1 && heads_q <= 65535 && heads_q % cache->heads == 0, PDH_EINVAL,
              "pdh_paged_attention: heads_q must be a multiple of the cache's heads");
  PDH_REQUIRE(window >= 1 && sinks >= 0, PDH_EINVAL, "pdh_paged_attention: window >= 1 and sinks >= 0");
  PDH_REQUIRE(std::isfinite(scale) && scale > 0.f, PDH_EINVAL, "pdh_paged_attention: scale must be finite and > 0");
  if (batch->rows == 0) return PDH_OK;
  PDH_REQUIRE(q && o && aligned16(q) && aligned16(o), PDH_EINVAL,
              "pdh_paged_attention: q and o must be 16-byte aligned");
  for (int64_t s : {q_st, q_sh, o_st, o_sh})
    PDH_REQUIRE(s >= 0 && s % 8 == 0, PDH_EINVAL, "pdh_paged_attention: strides must be multiples of 8 elements, >= 0");
  PagedAttn a{static_cast<const uint16_t*>(q), static_cast<uint16_t*>(o), lse, q_st, q_sh, o_st, o_sh, *cache, *batch,
              static_cast<int>(heads_q), static_cast<int>(heads_q / cache->heads),
              static_cast<int>(window < kMaxTokens ? window : kMaxTokens),
              static_cast<int>(sinks < kMaxTokens ? sinks : kMaxTokens), shift, zero_rest != 0,
              static_cast<int>(batch->width << shift), scale * kLog2e};
  const dim3 grid(static_cast<unsigned>(batch->rows), static_cast<unsigned>((heads_q + 3) / 4));
  by_kind(*cache, [&](auto t, auto d, auto bits) {
    paged_attn_rows<decltype(t), decltype(d)::value, decltype(bits)::value><<<grid, 256, 0, as_stream(stream)>>>(a);
  });
  return check_launch("pdh_paged_attention");
}
