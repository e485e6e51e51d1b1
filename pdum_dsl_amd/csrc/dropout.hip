// Dropout whose mask is a pure function of (seed, step, site, position), so
// that the backward pass recomputes it and nothing stores it:
//   y = [residual +] keep ? x * 65536 / (65536 - t) : 0,   t = floor(65536 p + 1/2)
//   keep = bits >= t, bits 16 random bits of the element.
// The bits come from Philox4x32-10 (J. Salmon, M. Moraes, R. Dror, D. Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", SC 2011): ten rounds of two
// 32 x 32 -> 64-bit products on a 128-bit counter under a 64-bit key. The key is the
// seed; the counter is (group low, group high, step low, site), group =
// row * ceil(cols / 8) + col / 8; the 128 bits serve the group's 8
// consecutive columns, 16 bits each, low halves first. The survivors' scale
// inverts the rate that t keeps exactly, so E[y] = x for every p although p
// is held to 2^-16. A dropped x counts for nothing, infinities and NaN
// included: it is selected away, not multiplied.
//
// The seed and the step are read from device memory: a captured graph draws a
// new mask at each replay once the caller has moved the step on.
//
// One lane serves one group: 16 bytes of a 16-bit row, 32 of an fp32 one.
// HBM-bound: 32768 x 4096 bf16 with a residual 127 us (6.3 TB/s), 8192 x 4096
// fp32 48 us (5.6). The generator's twenty 64-bit products a group take less
// than a group's bytes do. Loads and stores go past the caches: 8192 x 768 bf16
// 7.1 -> 6.2 us, with a residual 9.2 -> 8.3.
#include "common.h"

namespace pdh {
namespace {

constexpr uint32_t kPhiloxM0 = 0xD2511F53u, kPhiloxM1 = 0xCD9E8D57u;  // the paper's multipliers
constexpr uint32_t kPhiloxW0 = 0x9E3779B9u, kPhiloxW1 = 0xBB67AE85u;  // and key increments

__device__ __forceinline__ u32x4 philox4x32(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0,
                                            uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = static_cast<uint64_t>(c0) * kPhiloxM0, p1 = static_cast<uint64_t>(c2) * kPhiloxM1;
    c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(p1);
    c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(p0);
    k0 += kPhiloxW0;
    k1 += kPhiloxW1;
  }
  return u32x4{c0, c1, c2, c3};
}

struct DropoutArgs {
  const void* x;
  const void* res;
  void* y;
  const int64_t* rng;  // {seed, step}
  uint64_t group0;     // the first group of this launch
  uint32_t groups;     // groups of this launch (whole rows)
  uint32_t per_row;    // ceil(cols / 8)
  int cols;
  int64_t ldx, ldr, ldy;
  uint32_t threshold, site;
  float scale;
};

// Eight consecutive elements as fp32, at any alignment of the element type.
template <int DT>
__device__ __forceinline__ void load8(const void* p, float (&v)[8]) {
  if constexpr (DT == PDH_F32) {
    const f32x4u a = __builtin_nontemporal_load(static_cast<const f32x4u*>(p));
    const f32x4u b = __builtin_nontemporal_load(static_cast<const f32x4u*>(p) + 1);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = a[j], v[4 + j] = b[j];
  } else {
    const u32x4h w = __builtin_nontemporal_load(static_cast<const u32x4h*>(p));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint16_t e = static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)));
      v[j] = DT == PDH_BF16 ? bf16_to_f32(e) : f16_to_f32(e);
    }
  }
}

template <int DT>
__device__ __forceinline__ void store8(void* p, const float (&v)[8]) {
  if constexpr (DT == PDH_F32) {
    __builtin_nontemporal_store(f32x4u{v[0], v[1], v[2], v[3]}, static_cast<f32x4u*>(p));
    __builtin_nontemporal_store(f32x4u{v[4], v[5], v[6], v[7]}, static_cast<f32x4u*>(p) + 1);
  } else {
    u32x4h w;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = DT == PDH_BF16 ? pack2<__hip_bfloat16>(v[2 * j], v[2 * j + 1]) : pack2<_Float16>(v[2 * j], v[2 * j + 1]);
    __builtin_nontemporal_store(w, static_cast<u32x4h*>(p));
  }
}

template <int DT, bool RES>
__global__ __launch_bounds__(256) void dropout_rows(DropoutArgs a) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= a.groups) return;
  const uint32_t row = i / a.per_row, grp = i - row * a.per_row;
  const uint64_t g = a.group0 + i;
  constexpr int ES = DT == PDH_F32 ? 4 : 2;
  const int col = static_cast<int>(grp) * 8;
  const char* xp = static_cast<const char*>(a.x) + (static_cast<int64_t>(row) * a.ldx + col) * ES;
  const char* rp = RES ? static_cast<const char*>(a.res) + (static_cast<int64_t>(row) * a.ldr + col) * ES : nullptr;
  char* yp = static_cast<char*>(a.y) + (static_cast<int64_t>(row) * a.ldy + col) * ES;
  const uint64_t seed = static_cast<uint64_t>(a.rng[0]);
  const int left = a.cols - col;
  float v[8] = {}, r[8] = {};
  if (left >= 8) {
    load8<DT>(xp, v);
    if constexpr (RES) load8<DT>(rp, r);
  } else {
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (j < left) {
        v[j] = ld_dt<DT>(xp, j);
        if constexpr (RES) r[j] = ld_dt<DT>(rp, j);
      }
  }
  const u32x4 b = philox4x32(static_cast<uint32_t>(g), static_cast<uint32_t>(g >> 32),
                             static_cast<uint32_t>(a.rng[1]), a.site, static_cast<uint32_t>(seed),
                             static_cast<uint32_t>(seed >> 32));
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t bits = (j & 1) ? b[j >> 1] >> 16 : b[j >> 1] & 0xffffu;
    const float kept = bits >= a.threshold ? v[j] * a.scale : 0.f;
    v[j] = RES ? r[j] + kept : kept;
  }
  if (left >= 8) {
    store8<DT>(yp, v);
  } else {
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (j < left) st_dt<DT>(yp, j, v[j]);
  }
}

}  // namespace
}  // namespace pdh

using namespace pdh;

extern "C" int pdh_dropout(const void* x, const void* residual, void* y, int64_t rows, int64_t cols, int64_t ldx,
                           int64_t ldr, int64_t ldy, double p, const int64_t* rng, int64_t site, int dtype,
                           void* stream) {
  PDH_REQUIRE(dtype == PDH_F32 || dtype == PDH_BF16 || dtype == PDH_F16, PDH_EUNSUPPORTED, "pdh_dropout: dtype %d",
              dtype);
  PDH_REQUIRE(p >= 0.0 && p <= 1.0, PDH_EINVAL, "pdh_dropout: the rate p = %g must lie in [0, 1]",
              p);
  PDH_REQUIRE(site >= 0 && site <= int64_t{0xffffffff}, PDH_EINVAL, "pdh_dropout: site %lld is not 32 bits unsigned",
              (long long)site);
  PDH_REQUIRE(rows >= 0 && cols >= 1, PDH_EINVAL, "pdh_dropout: need rows >= 0 and cols >= 1 (got %lld, %lld)",
              (long long)rows, (long long)cols);
  PDH_REQUIRE(cols <= (int64_t{1} << 30), PDH_EINVAL, "pdh_dropout: rows longer than 2^30 elements");
  PDH_REQUIRE(ldx >= 0 && ldy >= cols && (!residual || ldr >= 0), PDH_EINVAL,
              "pdh_dropout: row strides must be >= 0, and y's >= cols (%lld)", (long long)cols);
  if (rows == 0) return PDH_OK;
  PDH_REQUIRE(x && y && rng, PDH_EINVAL, "pdh_dropout: null pointer");
  const int64_t es = dtype == PDH_F32 ? 4 : 2;
  const uint32_t threshold = static_cast<uint32_t>(p * 65536.0 + 0.5);
  DropoutArgs a{};
  a.rng = rng;
  a.per_row = static_cast<uint32_t>((cols + 7) / 8);
  a.cols = static_cast<int>(cols);
  a.ldx = ldx, a.ldr = ldr, a.ldy = ldy;
  a.threshold = threshold;
  a.site = static_cast<uint32_t>(site);
  a.scale = threshold >= 65536u ? 0.f : 65536.f / static_cast<float>(65536u - threshold);
  hipStream_t s = as_stream(stream);
  // launches of whole rows, under 2^31 groups each (the kernel counts them in 32 bits)
  const int64_t rows_max = (int64_t{1} << 31) / a.per_row - 1 > 0 ? (int64_t{1} << 31) / a.per_row - 1 : 1;
  for (int64_t r0 = 0; r0 < rows; r0 += rows_max) {
    const int64_t nr = rows - r0 < rows_max ? rows - r0 : rows_max;
    a.x = static_cast<const char*>(x) + r0 * ldx * es;
    a.res = residual ? static_cast<const char*>(residual) + r0 * ldr * es : nullptr;
    a.y = static_cast<char*>(y) + r0 * ldy * es;
    a.group0 = static_cast<uint64_t>(r0) * a.per_row;
    a.groups = static_cast<uint32_t>(nr * a.per_row);
    const dim3 grid((a.groups + 255u) / 256u);
#define PDH_DROP(DT)                                                  \
  do {                                                                \
    if (residual)                                                     \
      dropout_rows<DT, true><<<grid, 256, 0, s>>>(a);                 \
    else                                                              \
      dropout_rows<DT, false><<<grid, 256, 0, s>>>(a);                \
  } while (0)
    if (dtype == PDH_F32)
      PDH_DROP(PDH_F32);
    else if (dtype == PDH_BF16)
      PDH_DROP(PDH_BF16);
    else
      PDH_DROP(PDH_F16);
#undef PDH_DROP
    if (int rc = check_launch("pdh_dropout"); rc != PDH_OK) return rc;
  }
  return PDH_OK;
}
