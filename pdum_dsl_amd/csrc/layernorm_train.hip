// Layer norm in a training step: the forward that keeps its statistics and
// the backward with the weights' gradients.
//   mean = sum x / n, rstd = 1 / sqrt(sum (x - mean)^2 / n + eps), xh = (x - mean) rstd
//   y = xh gamma + beta
//   u = dy gamma, dx = rstd (u - mean(u) - xh mean(u xh)) [+ dres]
//   dgamma = sum_rows dy xh, dbeta = sum_rows dy
// Both are HBM-bound: the forward moves x and y, the backward x, dy, dx (and
// dres) once.
//
// A row is held in the registers of W waves (W = 1 up to 1024 columns, then 4,
// 8, 16), 16 values a lane, in chunks of 16 bytes; chunk i of lane l of wave w
// is chunk (i W + w) 64 + l of the row, so every load covers consecutive
// kilobytes. The hardware takes 16-byte accesses at any element's alignment,
// so rows of odd lengths and strides run the same path. Sums of a row: DPP rotations in
// 16-lane rows, four readlanes, LDS between waves.
//
// The backward's grid is fixed, a workgroup of eight waves (16 for the longest
// rows) on every compute unit: each walks its rows with the next row's loads in
// flight, keeps its columns' sums of dy xh and dy in registers and writes them
// once, fp32, to the workspace; a second kernel adds the workgroups' partial
// sums in order. No atomics: results repeat bit for bit. Two workgroups a unit
// hide no more latency and double the partial sums: 4096 x 4096 bf16 41.5 us
// against 34.8, 2048 x 8192 50 against 36.
//
// 8192 x 4096 fp32, the kernels' times in us: forward 38 (7.0 TB/s) on the same
// tensors again and again, which the caches hold in part, 50 (5.4) on six sets of
// tensors in turn; backward 71 (5.7) either way, 62 (6.4) right after the forward.
// In turn, 32768 x 768 bf16: 22 and 30; 8192 x 768: 7.3 and 11.9.
// Outputs leave past the caches (in the caches' place, forward in a step 66
// against 51, 8192 x 768 bf16 8.4 against 7.0). Loads go past them in the backward
// (through them, 75 against 71 in turn, but 64 against 71 on the same tensors) and
// through them in the forward (past them, 49 against 38 on the same tensors, and
// the backward after it 71 against 62).
//
// Rows of over 16384 columns, or of fewer than a chunk, take one workgroup a
// row in several passes of single elements, and column sums by a kernel of their
// own: right for any width, and far from the bytes' rate (forward and backward,
// 2048 x 20000 bf16 122 and 198 us, fp32 152 and 244; 65536 x 3 fp32 263 and 299).
#include "common.h"

namespace pdh {
namespace {

constexpr int kVals = 16;         // values of a row a lane holds
constexpr int kMaxCols = 16384;   // 16 waves x 64 lanes x kVals
constexpr int kBwdGroups = 256;   // workgroups of the backward: a compute unit each, and their partial sums
constexpr int64_t kFwdRows = int64_t{1} << 21;  // rows of one forward launch
constexpr int kLongGroups = 1 << 16;  // workgroups of the long rows' backward
constexpr int kSlices = 64;       // row slices of the long rows' column sums

template <int DT>
constexpr int es() {
  return DT == PDH_F32 ? 4 : 2;
}
template <int DT>
constexpr int vec() {  // elements of a 16-byte chunk
  return 16 / es<DT>();
}

// The sum over a wave, in every lane.
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float lane_of(float v, int l) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l));
}
__device__ __forceinline__ float wave_add(float v) {
  v = dpp_add<0x128>(v);  // row_ror:8, 4, 2, 1: every lane holds its 16-lane row's sum
  v = dpp_add<0x124>(v);
  v = dpp_add<0x122>(v);
  v = dpp_add<0x121>(v);
  return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}

template <int DT>
__device__ __forceinline__ float elem(u32x4 w, int j) {
  if constexpr (DT == PDH_F32) {
    return __uint_as_float(w[j]);
  } else {
    const uint16_t e = static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)));
    return DT == PDH_BF16 ? bf16_to_f32(e) : f16_to_f32(e);
  }
}

template <int DT>
__device__ __forceinline__ u32x4 pack_chunk(const float* v) {
  u32x4 w;
  if constexpr (DT == PDH_F32) {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = __float_as_uint(v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = DT == PDH_BF16 ? pack2<__hip_bfloat16>(v[2 * j], v[2 * j + 1]) : pack2<_Float16>(v[2 * j], v[2 * j + 1]);
  }
  return w;
}

// A lane's share of a row of at least V columns. Chunk i nominally starts at
// column col(i); the chunk that crosses the row's end is read (and written)
// as the row's last V columns, and so are the chunks past it, so that no load
// branches. Values j < skip(i) of a chunk are thus not this lane's: they count as
// zero in sums, and where the chunk crosses the end they are stored as the
// same values that their owner stores.
template <int DT, int W>
struct Share {
  static constexpr int V = vec<DT>(), CH = kVals / V;
  int c[CH], skip[CH];  // the columns read, and the values of each chunk that are another lane's

  __device__ __forceinline__ Share(int wave, int lane, int cols) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int col = ((i * W + wave) * 64 + lane) * V;
      c[i] = col < cols - V ? col : cols - V;
      skip[i] = col - c[i];
    }
  }
  __device__ __forceinline__ bool mine(int j) const { return j % V >= skip[j / V]; }
  // STREAM: past the caches, for a row that this launch reads once
  template <bool STREAM>
  __device__ __forceinline__ void load(const char* row, u32x4 (&w)[CH]) const {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const u32x4h* p = reinterpret_cast<const u32x4h*>(row + c[i] * es<DT>());
      w[i] = STREAM ? __builtin_bit_cast(u32x4, __builtin_nontemporal_load(p)) : __builtin_bit_cast(u32x4, *p);
    }
  }
  __device__ __forceinline__ void store(char* row, const float (&v)[kVals]) const {
#pragma unroll
    for (int i = 0; i < CH; ++i)
      if (skip[i] < V)
        __builtin_nontemporal_store(__builtin_bit_cast(u32x4h, pack_chunk<DT>(v + i * V)),
                                    reinterpret_cast<u32x4h*>(row + c[i] * es<DT>()));
  }
};

// Sums over the W waves of a row (two values at once); `sh` holds 2 x W floats
// of this reduction alone, so one barrier suffices.
template <int W>
__device__ __forceinline__ void row_add2(float& a, float& b, float* sh, int wave, int lane) {
  a = wave_add(a);
  b = wave_add(b);
  if constexpr (W > 1) {
    if (lane == 0) sh[wave] = a, sh[W + wave] = b;
    __syncthreads();
    a = 0.f, b = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) a += sh[i], b += sh[W + i];
  }
}
template <int W>
__device__ __forceinline__ float row_add(float a, float* sh, int wave, int lane) {
  a = wave_add(a);
  if constexpr (W > 1) {
    if (lane == 0) sh[wave] = a;
    __syncthreads();
    a = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) a += sh[i];
  }
  return a;
}

struct NormArgs {
  const void* x;
  const void* gamma;
  const void* beta;
  void* y;
  float* mean;
  float* rstd;
  int64_t rows, ldx, ldy;
  int cols;
  float eps;
};

// R rows a workgroup, W waves a row.
template <int DT, int W, int R>
__global__ __launch_bounds__(64 * W * R) void norm_fwd(NormArgs a) {
  using S = Share<DT, W>;
  __shared__ float sh[2 * W];
  const int lane = threadIdx.x & 63, w = wave_id(), wave = w % W;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * R + w / W;
  if (W == 1 && row >= a.rows) return;  // W > 1 has R = 1: the grid is the rows
  const S sh_of(wave, lane, a.cols);
  u32x4 raw[S::CH], gw[S::CH], bw[S::CH];
  sh_of.template load<false>(static_cast<const char*>(a.x) + row * a.ldx * es<DT>(), raw);
  if (a.gamma) sh_of.template load<false>(static_cast<const char*>(a.gamma), gw);
  if (a.beta) sh_of.template load<false>(static_cast<const char*>(a.beta), bw);
  float v[kVals], s = 0.f, ss = 0.f;
#pragma unroll
  for (int j = 0; j < kVals; ++j) {
    v[j] = elem<DT>(raw[j / S::V], j % S::V);
    s += sh_of.mine(j) ? v[j] : 0.f;
  }
  // divided, not multiplied by 1 / n: the mean of equal values whose sum is exact is that value
  const float n = static_cast<float>(a.cols), mean = row_add<W>(s, sh, wave, lane) / n;
#pragma unroll
  for (int j = 0; j < kVals; ++j) {
    v[j] -= mean;
    ss += sh_of.mine(j) ? v[j] * v[j] : 0.f;
  }
  const float rstd = 1.f / sqrtf(row_add<W>(ss, sh + W, wave, lane) / n + a.eps);
#pragma unroll
  for (int j = 0; j < kVals; ++j) {
    v[j] *= rstd;
    if (a.gamma) v[j] *= elem<DT>(gw[j / S::V], j % S::V);
    if (a.beta) v[j] += elem<DT>(bw[j / S::V], j % S::V);
  }
  sh_of.store(static_cast<char*>(a.y) + row * a.ldy * es<DT>(), v);
  if (lane == 0 && wave == 0) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
}

struct NormGradArgs {
  const void* x;
  const void* dy;
  const void* dres;
  const void* gamma;
  const float* mean;
  const float* rstd;
  void* dx;
  float* part;  // [groups][2][cols]: a workgroup's sums of dy xh and of dy
  int64_t rows, ldx, lddy, lddres, lddx;
  int cols;
};

// R rows at a time in a workgroup, W waves a row; the workgroup's rows are
// blockIdx + gridDim * (0, 1, ...), in units of R.
template <int DT, int W, int R, bool AFFINE>
__global__ __launch_bounds__(64 * W * R) void norm_bwd(NormGradArgs a) {
  using S = Share<DT, W>;
  constexpr int CH = S::CH, V = S::V;
  // two reductions' worth, used in turn: a wave writes one while a slow one still reads the other
  __shared__ float sh[R][2][2 * W];
  __shared__ float acc_sh[AFFINE && R > 1 ? R * 64 * W * kVals : 1];
  const int lane = threadIdx.x & 63, w = wave_id(), wave = w % W, slot = w / W;
  const int64_t step = static_cast<int64_t>(gridDim.x) * R;
  int64_t row = static_cast<int64_t>(blockIdx.x) * R + slot;
  const float inv_n = 1.f / static_cast<float>(a.cols);
  const S own(wave, lane, a.cols);
  u32x4 gw[CH], xw[CH], yw[CH], rw[CH];
  float ag[kVals] = {}, ab[kVals] = {}, mean = 0.f, rstd = 0.f;
  if (AFFINE) own.template load<false>(static_cast<const char*>(a.gamma), gw);
  auto fetch = [&](int64_t r) __attribute__((always_inline)) {
    own.template load<true>(static_cast<const char*>(a.x) + r * a.ldx * es<DT>(), xw);
    own.template load<true>(static_cast<const char*>(a.dy) + r * a.lddy * es<DT>(), yw);
    if (a.dres) own.template load<true>(static_cast<const char*>(a.dres) + r * a.lddres * es<DT>(), rw);
    mean = a.mean[r];
    rstd = a.rstd[r];
  };
  // 16 waves leave 128 registers a lane, too few for the next row's loads
  constexpr bool AHEAD = W < 16;
  if (AHEAD && row < a.rows) fetch(row);
  int turn = 0;
  // with more than one wave a row the slots meet at barriers: all run the first one's rounds
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * R; first < a.rows; first += step, row += step, turn ^= 1) {
    const bool live = R == 1 || row < a.rows;
    if (W == 1 && !live) break;
    if (!AHEAD && live) fetch(row);
    float xh[kVals], u[kVals], o[kVals], su = 0.f, sux = 0.f;
    const float rs = rstd;
#pragma unroll
    for (int j = 0; j < kVals; ++j) {
      const float d = elem<DT>(yw[j / V], j % V);
      xh[j] = (elem<DT>(xw[j / V], j % V) - mean) * rs;
      u[j] = AFFINE ? d * elem<DT>(gw[j / V], j % V) : d;
      o[j] = a.dres ? elem<DT>(rw[j / V], j % V) : 0.f;
      if (AFFINE && live) {  // another lane's values are left out of the store below
        ag[j] += d * xh[j];
        ab[j] += d;
      }
      su += own.mine(j) ? u[j] : 0.f;
      sux += own.mine(j) ? u[j] * xh[j] : 0.f;
    }
    const int64_t next = row + step;
    if (AHEAD && next < a.rows) fetch(next);
    row_add2<W>(su, sux, sh[slot][turn], wave, lane);
    const float c1 = su * inv_n, c2 = sux * inv_n;
#pragma unroll
    for (int j = 0; j < kVals; ++j) o[j] += rs * (u[j] - c1 - xh[j] * c2);
    if (live) own.store(static_cast<char*>(a.dx) + row * a.lddx * es<DT>(), o);
  }
  if constexpr (AFFINE) {
    float* part = a.part + static_cast<int64_t>(blockIdx.x) * 2 * a.cols;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      float(&v)[kVals] = which ? ab : ag;
      if constexpr (R > 1) {  // the row slots' sums, added in order
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kVals; ++j) acc_sh[(slot * W + wave) * 64 * kVals + j * 64 + lane] = v[j];
        __syncthreads();
        if (slot != 0) continue;
#pragma unroll
        for (int j = 0; j < kVals; ++j) {
          float s = 0.f;
          for (int q = 0; q < R; ++q) s += acc_sh[(q * W + wave) * 64 * kVals + j * 64 + lane];
          v[j] = s;
        }
      }
#pragma unroll
      for (int j = 0; j < kVals; ++j)
        if (own.mine(j)) part[static_cast<int64_t>(which) * a.cols + own.c[j / V] + j % V] = v[j];
    }
  }
}

// dgamma / dbeta = the sums over `n` partial rows [n][2][cols], in a fixed
// order: 16 columns of one of the two a workgroup, 64 lanes a column with
// four loads in flight each (768 columns, 256 parts: 3.5-4 us; 512 parts, of an
// earlier grid, took 4 so and 20 with 8 lanes a column on 48 workgroups, a chain
// of loads).
template <int DT>
__global__ __launch_bounds__(1024) void norm_weights(const float* __restrict__ part, int n, int64_t cols, void* dgamma,
                                                     void* dbeta) {
  __shared__ float sh[64][17];
  const int c16 = threadIdx.x & 15, q = threadIdx.x >> 4;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 16 + c16;
  const int which = blockIdx.y;
  float s = 0.f;
  if (c < cols) {
    const float* p = part + which * cols + c;
    for (int i = q; i < n; i += 256) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = i + 64 * j < n ? p[static_cast<int64_t>(i + 64 * j) * 2 * cols] : 0.f;
      s += (v[0] + v[1]) + (v[2] + v[3]);
    }
  }
  sh[q][c16] = s;
  __syncthreads();
  if (threadIdx.x < 256) {  // four lanes' sums each, then the sixteen
    const int r = threadIdx.x >> 4;
    s = (sh[4 * r][c16] + sh[4 * r + 1][c16]) + (sh[4 * r + 2][c16] + sh[4 * r + 3][c16]);
  }
  __syncthreads();
  if (threadIdx.x < 256) sh[threadIdx.x >> 4][c16] = s;
  __syncthreads();
  if (threadIdx.x < 16 && c < cols) {
    s = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) s += sh[r][c16];
    st_dt<DT>(which ? dbeta : dgamma, c, s);
  }
}

// ---- rows that no wave holds: one workgroup a row, several passes ----

__device__ __forceinline__ float group_add(float v, float* sh) {
  v = wave_add(v);
  __syncthreads();  // the last reduction's reads are over
  if ((threadIdx.x & 63) == 0) sh[wave_id()] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < static_cast<int>(blockDim.x >> 6); ++i) s += sh[i];
  return s;
}

template <int DT>
__global__ __launch_bounds__(1024) void norm_fwd_long(NormArgs a) {
  __shared__ float sh[16];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const char* x = static_cast<const char*>(a.x) + row * a.ldx * es<DT>();
    char* y = static_cast<char*>(a.y) + row * a.ldy * es<DT>();
    float s = 0.f, ss = 0.f;
    for (int c = threadIdx.x; c < a.cols; c += 1024) s += ld_dt<DT>(x, c);
    const float mean = group_add(s, sh) / static_cast<float>(a.cols);
    for (int c = threadIdx.x; c < a.cols; c += 1024) {
      const float d = ld_dt<DT>(x, c) - mean;
      ss += d * d;
    }
    const float rstd = 1.f / sqrtf(group_add(ss, sh) / static_cast<float>(a.cols) + a.eps);
    for (int c = threadIdx.x; c < a.cols; c += 1024) {
      float o = (ld_dt<DT>(x, c) - mean) * rstd;
      if (a.gamma) o *= ld_dt<DT>(a.gamma, c);
      if (a.beta) o += ld_dt<DT>(a.beta, c);
      st_dt<DT>(y, c, o);
    }
    if (threadIdx.x == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

template <int DT>
__global__ __launch_bounds__(1024) void norm_bwd_long(NormGradArgs a) {
  __shared__ float sh[16];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const char* x = static_cast<const char*>(a.x) + row * a.ldx * es<DT>();
    const char* dy = static_cast<const char*>(a.dy) + row * a.lddy * es<DT>();
    const char* dres = a.dres ? static_cast<const char*>(a.dres) + row * a.lddres * es<DT>() : nullptr;
    char* dx = static_cast<char*>(a.dx) + row * a.lddx * es<DT>();
    const float mean = a.mean[row], rstd = a.rstd[row];
    auto u_at = [&](int c) {
      const float d = ld_dt<DT>(dy, c);
      return a.gamma ? d * ld_dt<DT>(a.gamma, c) : d;
    };
    float su = 0.f, sux = 0.f;
    for (int c = threadIdx.x; c < a.cols; c += 1024) {
      const float u = u_at(c);
      su += u;
      sux += u * ((ld_dt<DT>(x, c) - mean) * rstd);
    }
    const float c1 = group_add(su, sh) / static_cast<float>(a.cols);
    const float c2 = group_add(sux, sh) / static_cast<float>(a.cols);
    for (int c = threadIdx.x; c < a.cols; c += 1024) {
      const float xh = (ld_dt<DT>(x, c) - mean) * rstd;
      const float o = rstd * (u_at(c) - c1 - xh * c2);
      st_dt<DT>(dx, c, dres ? o + ld_dt<DT>(dres, c) : o);
    }
  }
}

// part[slice][2][cols] = sums over the slice's rows of dy xh and dy: 64
// columns a workgroup, four rows at a time.
template <int DT>
__global__ __launch_bounds__(256) void norm_cols_long(NormGradArgs a) {
  __shared__ float sh[2][4][64];
  const int lane = threadIdx.x & 63, q = threadIdx.x >> 6;
  const int c = static_cast<int>(blockIdx.x) * 64 + lane;
  const int64_t slice = blockIdx.y, n = gridDim.y;
  const int64_t r0 = a.rows * slice / n, r1 = a.rows * (slice + 1) / n;
  float g = 0.f, b = 0.f;
  if (c < a.cols)
    for (int64_t r = r0 + q; r < r1; r += 4) {
      const float d = ld_dt<DT>(static_cast<const char*>(a.dy) + r * a.lddy * es<DT>(), c);
      g += d * ((ld_dt<DT>(static_cast<const char*>(a.x) + r * a.ldx * es<DT>(), c) - a.mean[r]) * a.rstd[r]);
      b += d;
    }
  sh[0][q][lane] = g;
  sh[1][q][lane] = b;
  __syncthreads();
  if (q < 2 && c < a.cols)
    a.part[(slice * 2 + q) * a.cols + c] = (sh[q][0][lane] + sh[q][1][lane]) + (sh[q][2][lane] + sh[q][3][lane]);
}

template <int DT>
void launch_fwd(const NormArgs& all, hipStream_t s) {
  if (all.rows > kFwdRows) {  // a launch holds under 2^32 threads
    for (int64_t r0 = 0; r0 < all.rows; r0 += kFwdRows) {
      NormArgs a = all;
      a.rows = all.rows - r0 < kFwdRows ? all.rows - r0 : kFwdRows;
      a.x = static_cast<const char*>(all.x) + r0 * all.ldx * es<DT>();
      a.y = static_cast<char*>(all.y) + r0 * all.ldy * es<DT>();
      a.mean = all.mean + r0;
      a.rstd = all.rstd + r0;
      launch_fwd<DT>(a, s);
    }
    return;
  }
  const NormArgs& a = all;
  const unsigned rows = static_cast<unsigned>(a.rows);
  if (a.cols < vec<DT>() || a.cols > kMaxCols)
    norm_fwd_long<DT><<<dim3(rows), 1024, 0, s>>>(a);
  else if (a.cols <= 1024)
    norm_fwd<DT, 1, 4><<<dim3((rows + 3) / 4), 256, 0, s>>>(a);
  else if (a.cols <= 4096)
    norm_fwd<DT, 4, 1><<<dim3(rows), 256, 0, s>>>(a);
  else if (a.cols <= 8192)
    norm_fwd<DT, 8, 1><<<dim3(rows), 512, 0, s>>>(a);
  else
    norm_fwd<DT, 16, 1><<<dim3(rows), 1024, 0, s>>>(a);
}

bool long_rows(int64_t cols, int dtype) { return cols > kMaxCols || cols < (dtype == PDH_F32 ? 4 : 8); }
int bwd_rows(int64_t cols) { return cols <= 1024 ? 8 : cols <= 4096 ? 2 : 1; }  // rows a workgroup takes at a time

// Partial rows of the weights' gradients.
int64_t bwd_parts(int64_t rows, int64_t cols, int dtype) {
  if (long_rows(cols, dtype)) return rows < kSlices ? rows : kSlices;
  const int64_t per = bwd_rows(cols), g = (rows + per - 1) / per;
  return g < kBwdGroups ? g : kBwdGroups;
}

template <int DT, bool AFFINE>
void launch_bwd(const NormGradArgs& a, unsigned groups, hipStream_t s) {
  if (long_rows(a.cols, DT)) {
    // the column sums first: dx may take x's or dy's place
    if (AFFINE) norm_cols_long<DT><<<dim3((a.cols + 63) / 64, groups), 256, 0, s>>>(a);
    norm_bwd_long<DT><<<dim3(static_cast<unsigned>(a.rows < kLongGroups ? a.rows : kLongGroups)), 1024, 0, s>>>(a);
  } else if (a.cols <= 1024)
    norm_bwd<DT, 1, 8, AFFINE><<<dim3(groups), 512, 0, s>>>(a);
  else if (a.cols <= 4096)
    norm_bwd<DT, 4, 2, AFFINE><<<dim3(groups), 512, 0, s>>>(a);
  else if (a.cols <= 8192)
    norm_bwd<DT, 8, 1, AFFINE><<<dim3(groups), 512, 0, s>>>(a);
  else
    norm_bwd<DT, 16, 1, AFFINE><<<dim3(groups), 1024, 0, s>>>(a);
}

template <int DT>
int run_bwd(const NormGradArgs& a, void* dgamma, void* dbeta, hipStream_t s) {
  const int64_t parts = bwd_parts(a.rows, a.cols, DT);
  if (a.rows > 0) {
    if (dgamma)
      launch_bwd<DT, true>(a, static_cast<unsigned>(parts), s);
    else
      launch_bwd<DT, false>(a, static_cast<unsigned>(parts), s);
    if (int rc = check_launch("pdh_layernorm_bwd"); rc != PDH_OK) return rc;
  }
  if (dgamma) {
    norm_weights<DT><<<dim3(static_cast<unsigned>((a.cols + 15) / 16), 2), 1024, 0, s>>>(
        a.part, static_cast<int>(parts), a.cols, dgamma, dbeta);
    return check_launch("pdh_layernorm_bwd (weights)");
  }
  return PDH_OK;
}

int check_shape(const char* fn, int64_t rows, int64_t cols, int dtype) {
  PDH_REQUIRE(dtype == PDH_F32 || dtype == PDH_BF16 || dtype == PDH_F16, PDH_EUNSUPPORTED, "%s: dtype %d", fn, dtype);
  PDH_REQUIRE(rows >= 0 && cols >= 1, PDH_EINVAL, "%s: need rows >= 0 and cols >= 1 (got %lld, %lld)", fn,
              (long long)rows, (long long)cols);
  PDH_REQUIRE(rows <= INT32_MAX, PDH_EINVAL, "%s: too many rows", fn);
  PDH_REQUIRE(cols <= (int64_t{1} << 28), PDH_EINVAL, "%s: rows longer than 2^28 elements", fn);
  return PDH_OK;
}

}  // namespace
}  // namespace pdh

using namespace pdh;

extern "C" int pdh_layernorm_fwd(const void* x, const void* gamma, const void* beta, void* y, float* mean, float* rstd,
                                 int64_t rows, int64_t cols, int64_t ldx, int64_t ldy, float eps, int dtype,
                                 void* stream) {
  if (int rc = check_shape("pdh_layernorm_fwd", rows, cols, dtype); rc != PDH_OK) return rc;
  PDH_REQUIRE(ldx >= 0 && ldy >= cols, PDH_EINVAL,
              "pdh_layernorm_fwd: row strides (%lld, %lld) must be >= 0 and >= cols (%lld)", (long long)ldx,
              (long long)ldy, (long long)cols);
  PDH_REQUIRE(eps >= 0.f, PDH_EINVAL, "pdh_layernorm_fwd: eps must be >= 0");
  if (rows == 0) return PDH_OK;
  PDH_REQUIRE(x && y && mean && rstd, PDH_EINVAL, "pdh_layernorm_fwd: null pointer");
  const NormArgs a{x, gamma, beta, y, mean, rstd, rows, ldx, ldy, static_cast<int>(cols), eps};
  hipStream_t s = as_stream(stream);
  if (dtype == PDH_F32)
    launch_fwd<PDH_F32>(a, s);
  else if (dtype == PDH_BF16)
    launch_fwd<PDH_BF16>(a, s);
  else
    launch_fwd<PDH_F16>(a, s);
  return check_launch("pdh_layernorm_fwd");
}

extern "C" size_t pdh_layernorm_bwd_workspace(int64_t rows, int64_t cols, int dtype) {
  if (rows < 1 || cols < 1) return 0;
  return static_cast<size_t>(bwd_parts(rows, cols, dtype)) * 2 * static_cast<size_t>(cols) * sizeof(float);
}

extern "C" int pdh_layernorm_bwd(const void* x, const void* dy, const void* dres, const void* gamma, const float* mean,
                                 const float* rstd, void* dx, void* dgamma, void* dbeta, int64_t rows, int64_t cols,
                                 int64_t ldx, int64_t lddy, int64_t lddres, int64_t lddx, int dtype, void* ws,
                                 size_t ws_bytes, void* stream) {
  if (int rc = check_shape("pdh_layernorm_bwd", rows, cols, dtype); rc != PDH_OK) return rc;
  PDH_REQUIRE(ldx >= 0 && lddy >= 0 && lddx >= cols && (!dres || lddres >= 0), PDH_EINVAL,
              "pdh_layernorm_bwd: row strides must be >= 0, and dx's >= cols (%lld)", (long long)cols);
  PDH_REQUIRE(!dgamma == !dbeta && !dgamma == !gamma, PDH_EINVAL,
              "pdh_layernorm_bwd: gamma, dgamma and dbeta come together");
  PDH_REQUIRE(rows == 0 || (x && dy && mean && rstd && dx), PDH_EINVAL, "pdh_layernorm_bwd: null pointer");
  const size_t need = dgamma ? pdh_layernorm_bwd_workspace(rows, cols, dtype) : 0;
  PDH_REQUIRE(need == 0 || (ws && ws_bytes >= need), PDH_EINVAL,
              "pdh_layernorm_bwd: the workspace holds %zu bytes, %zu are needed", ws ? ws_bytes : size_t{0}, need);
  const NormGradArgs a{x,  dy,   dres, gamma, mean, rstd, dx, static_cast<float*>(ws), rows,
                       ldx, lddy, lddres, lddx, static_cast<int>(cols)};
  hipStream_t s = as_stream(stream);
  if (dtype == PDH_F32) return run_bwd<PDH_F32>(a, dgamma, dbeta, s);
  if (dtype == PDH_BF16) return run_bwd<PDH_BF16>(a, dgamma, dbeta, s);
  return run_bwd<PDH_F16>(a, dgamma, dbeta, s);
}
