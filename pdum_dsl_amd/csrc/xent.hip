// Softmax cross entropy of a linear head over a large vocabulary, and its
// gradient, without the logits in memory:
//   z[n, v] = sum_d x[n, d] w[v, d], lse[n] = log sum_v exp z[n, v]
//   loss[n] = lse[n] - z[n, target[n]]
//   dz[n, v] = dloss[n] (exp(z[n, v] - lse[n]) - [v = target[n]])
//   dx = dz w, dw = dz^T x
// Forward: one product kernel whose tiles of z stay in accumulators; each wave
// leaves the maximum and the sum of exponentials of its vocabulary strip of
// every token, and the target's logit where it holds it; a second kernel joins
// the strips. Backward: the vocabulary in pieces; for each the same product again,
// dz of the piece stored in 16 bits (2 bytes a token and entry, fp32's three terms
// 6; 1 GiB at the most, or 256 entries), then dw's rows of the piece and the
// piece's part of dx as two more products. dx's parts over slices of the
// vocabulary (and dw's over slices of the tokens, where its tiles are few) are
// fp32 and added in order: no atomics, results repeat.
//
// All three products run one tile loop (xent_tile): 256 x 128 tiles, four waves
// of 128 x 64, v_mfma_f32_32x32x16, accumulators m along registers and n along
// lanes; 64-deep k tiles by direct loads, whole 128-byte lines of a
// k-contiguous operand. An operand is k-contiguous or has its rows (m or n)
// contiguous, read transposed by ds_read_b64_tr_b16, so nothing is transposed
// in memory. The m rows are dealt to the matrix instruction's rows
// so that a lane's 16 accumulators are 16 consecutive m: whole vocabulary runs
// for the softmax, 32 bytes of an output row for the stores.
//
// dz is rounded to the storage type, as the probabilities of a 16-bit
// attention are: a relative 2^-8 (2^-11) of each term at most, independent from
// term to term, as the rounding of the 16-bit gradients they sum to. It is taken
// over the largest |dloss|, which the products' fp32 results are multiplied by:
// a mean's equal weights 1 / tokens would give every target's entry the same
// rounding error, which no sum averages out (0.38% of the gradient at 7780
// live tokens, 0.17% so, what the output's own rounding leaves); fp16 takes it
// times 2^14 on top, or small probabilities would fall below its range (its spacing
// is then 2^-38 of that weight at the finest), and
// fp32's terms stay clear of subnormal values for weights of any size. fp32 operands are split into three bf16 terms
// and the six cross products above 2^-24 are summed, smallest first.
//
// Bound by the matrix pipe at the clock that the power limit leaves it (49-68%
// busy at 1.55-1.9 GHz in every large product). Forward and backward in us, and
// the rate of the products run (z's again among the backward's): 8192 x 768 x
// 50257 bf16 554 (1141 TF/s) and 1903 (997), 4096 x 4096 x 50257 1390 (1213) and
// 4390 (1153), 1024 x 768 x 50257 fp32 445 (1066, of bf16 products) and 1385
// (1027); a library's bf16 product of 16384 cubed runs at 1338, of 8192 cubed at
// 1088. Small ones are bound by steps of 0.5 us a 64-deep k tile on few
// compute units (100 x 768 x 5003: 9 us of product, 4 of join).
#include "common.h"

#include <algorithm>

namespace pdh {
namespace {

constexpr int kBK = 64;  // k depth of a tile: a 128-byte line of a k-contiguous operand
constexpr uint32_t kOOB = 0x80000000u;  // past every buffer's extent: reads as zero
// fp32: the products of bf16 terms, in order of growing size: terms (0, 2) (2, 0)
// (1, 1) (0, 1) (1, 0) (0, 0) of (a, b), two bits each
constexpr int kPairs = 6, kPairA = 0x0118, kPairB = 0x0052;

// A 16-bit operand: rows of `pitch` bytes; k-contiguous (a row holds one m's or
// n's k values) or not (a row holds one k's m or n values). fp32 operands lie
// as three planes of bf16 terms, `plane` bytes apart.
struct Operand {
  const char* p;
  int64_t pitch, plane;
};

struct TileArgs {
  Operand a, b;
  int m, n, k;  // extents
  int tiles_m, tiles_n, slices;
  int kslice;   // k columns of a slice (a multiple of kBK)
  int group;    // n tiles that neighbouring workgroups share an m tile across
};

// Two runs of workgroups in one launch: `first` ids, then `second`. Workgroups
// go to the XCDs in turn (blockIdx % 8); each XCD takes a contiguous eighth of
// either run, so that its neighbours share operand panels in its L2. Returns
// the id in its run, or -1 for a workgroup past its end.
__device__ __forceinline__ int run_id(uint32_t first, uint32_t second, bool& in_second) {
  const uint32_t xcd = blockIdx.x & 7, pos = blockIdx.x >> 3, c1 = (first + 7) / 8, c2 = (second + 7) / 8;
  in_second = pos >= c1;
  const uint32_t id = in_second ? xcd * c2 + (pos - c1) : xcd * c1 + pos;
  return (in_second ? pos - c1 < c2 && id < second : id < first) ? static_cast<int>(id) : -1;
}
dim3 run_grid(int64_t first, int64_t second) {
  return dim3(static_cast<unsigned>(((first + 7) / 8 + (second + 7) / 8) * 8));
}

// Tile `id`: slices outermost, then groups of n tiles, m, the group's n tiles.
struct Tile {
  int m, n, slice;
};
__device__ __forceinline__ Tile tile_of(const TileArgs& a, uint32_t id) {
  const uint32_t per = static_cast<uint32_t>(a.tiles_m) * a.tiles_n;
  Tile t;
  t.slice = static_cast<int>(id / per);
  id -= t.slice * per;
  const uint32_t gsize = static_cast<uint32_t>(a.group) * a.tiles_m, g = id / gsize, rem = id - g * gsize;
  const uint32_t n0 = g * a.group, gn = min(static_cast<uint32_t>(a.tiles_n) - n0, static_cast<uint32_t>(a.group));
  t.m = static_cast<int>(rem / gn);
  t.n = static_cast<int>(n0 + rem % gn);
  return t;
}

// A workgroup: WM x WN waves of 32 TM (m) x 32 TN (n). NS 0: LDS holds two k
// tiles of a and one of b (80 KB for 256 x 128, two workgroups a compute unit);
// otherwise NS k tiles of both.
template <int WM_, int WN_, int TM_, int TN_, int NS_>
struct Config {
  static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_, NS = NS_;
  static constexpr int NW = WM * WN, BM = 32 * TM * WM, BN = 32 * TN * WN, THREADS = 64 * NW;
  static constexpr int LDS_A = BM * kBK * 2, LDS_B = BN * kBK * 2;
  static constexpr int LDS = NS ? NS * (LDS_A + LDS_B) : 2 * LDS_A + LDS_B;
};

// One operand's side of the loop. R: its rows in the tile (BM or BN), T: a
// wave's 32-row blocks; KC: k-contiguous; PERM: rows dealt as described above (the m side).
template <int R, int T, int NW, bool KC, bool PERM>
struct Side {
  static constexpr int BLOCKS = R * kBK * 2 / 1024 / NW;  // direct loads (1 KB) per wave and k tile
  static constexpr int KS = kBK / 16;                     // products deep
  static constexpr int PITCH = KC ? kBK * 2 : R * 2;      // LDS bytes of a row (rows contiguous: of a k row)
  static constexpr int SLOTS = PITCH / 16, ROWS = 64 / SLOTS;  // its 16-byte slots; rows a direct load covers
  static_assert(BLOCKS * 1024 * NW == R * kBK * 2 && NW % 4 == 0, "whole direct loads");
  uint32_t voff, vtail;  // the lane's byte offset in a direct load; the same in a ragged last k tile
  uint32_t pitch;
  int read[KC ? KS : T];  // LDS offsets of the lane's fragments: block 0's, or step 0's, without the tr read's second half

  // 16-byte slots are XOR-swizzled so that neither the b128 reads (16 lanes a cycle, the
  // quads of one parity in each half wave) nor the tr reads (32 lanes) meet a bank twice.
  __device__ __forceinline__ static int swz(int row) {
    if constexpr (KC) return (row & 7) ^ ((row >> 3) & 1);
    return R >= 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1);
  }

  __device__ __forceinline__ Side(const Operand& o, int wq, int lane, int w, int ktail) {
    pitch = static_cast<uint32_t>(o.pitch);
    // this wave's direct loads are w, w + NW, ...: their rows agree as far as swz looks
    const int row = lane / SLOTS, chunk = (lane % SLOTS) ^ swz(ROWS * w + row);
    voff = row * pitch + (chunk << 4);
    vtail = !KC || 8 * chunk < ktail ? voff : kOOB;  // (k rows past the end lie past the extent)
    if constexpr (KC) {  // a block is 32 rows on: the same swizzle
      const int r = lane & 31, g = lane >> 5;
      const int at = 32 * wq * T + (PERM ? 16 * ((r >> 2) & 1) + 4 * (r >> 3) + (r & 3) : r);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) read[ks] = at * PITCH + (((2 * ks + g) ^ swz(at)) << 4);
    } else {  // a step is 16 k rows on: the same swizzle
      const int G = lane >> 4, i4 = (lane >> 2) & 3, q = 4 * (G & 1) + (lane & 3);
      const int kr = 8 * (G >> 1) + i4;
#pragma unroll
      for (int t = 0; t < T; ++t) {
        const int col = 32 * (wq * T + t) + (PERM ? 16 * (q & 1) + 4 * (q >> 1) : 4 * q);
        read[t] = kr * PITCH + (((col >> 3) ^ swz(kr)) << 4) + ((col >> 2) & 1) * 8;
      }
    }
  }

  // Direct loads of k columns k0 .. k0 + 63 of rows r0 .. r0 + R - 1 (`rows` of them in the operand, `k` columns).
  __device__ __forceinline__ void fetch(const Operand& o, int64_t plane, int64_t r0, int rows, int64_t k0, int64_t k,
                                        uint32_t lds, int w) const {
    const char* base;
    uint32_t extent;
    const bool last = k - k0 < kBK;
    const int64_t nr = rows - r0 < R ? rows - r0 : R, nk = last ? k - k0 : kBK;
    if constexpr (KC) {
      base = o.p + plane * o.plane + r0 * o.pitch + k0 * 2;
      extent = static_cast<uint32_t>((nr - 1) * o.pitch + ((nk * 2 + 15) & ~int64_t{15}));
    } else {
      base = o.p + plane * o.plane + k0 * o.pitch + r0 * 2;
      extent = static_cast<uint32_t>((nk - 1) * o.pitch + ((nr * 2 + 15) & ~int64_t{15}));
    }
    const rsrc_t rs = make_rsrc(base, extent);
    const uint32_t v = last ? vtail : voff;
#pragma unroll
    for (int i = 0; i < BLOCKS; ++i) {
      const int blk = NW * i + w;
      dma16_at(rs, lds + blk * 1024, v, static_cast<uint32_t>(ROWS * blk) * pitch);
    }
  }

  __device__ __forceinline__ u32x4 frag(const unsigned char* tile, int t, int ks) const {
    if constexpr (KC) {
      return *reinterpret_cast<const u32x4*>(tile + read[ks] + 32 * t * PITCH);
    } else {
      const unsigned char* p = tile + read[t] + 16 * ks * PITCH;
      const u32x2 lo = ds_read_tr16(p), hi = ds_read_tr16(p + 4 * PITCH);
      return u32x4{lo.x, lo.y, hi.x, hi.y};
    }
  }
};

// acc = the products of a tile over k columns [k0, k1): accumulator i of
// (tm, tn) is m = m0 + 32 (wm TM + tm) + 16 (lane / 32) + i, n = n0 + 32 (wn TN + tn) + lane % 32.
// SPLIT: the operands are planes of bf16 terms, every k tile runs kPairs times.
//
// A k tile's b fragments go to registers first, so b needs one buffer: a
// second barrier frees it for the next tile's loads, which, with a's, are in
// flight under this tile's products. 64-deep tiles in two such workgroups a
// compute unit against 32-deep ones three deep in LDS: a k-contiguous operand's
// 64-byte rows cost every line two requests (fwd 8192 x 768 x 50257: 630 us,
// this 544; 4096 x 4096: 1640, 1420, the matrix pipe 66% busy at the 1.62 GHz
// that the part then holds); 256 x 256 tiles of eight waves, one workgroup a
// unit: 610, 1450; fragments read a step ahead across the barrier: no change.
// Workgroups that walk over their tiles, the next one's first loads under the
// last products, fall out of step, and neighbours no longer find each other's
// panels in L2: 1420 -> 1515, 560 -> 593 (so does any other staggering).
template <int DT, typename C, bool KA, bool KB, bool SPLIT>
__device__ __forceinline__ void xent_tile(const TileArgs& a, unsigned char* smem, f32x16 (&acc)[C::TM][C::TN], int m0,
                                          int n0, int64_t k0, int64_t k1) {
  constexpr int TM = C::TM, TN = C::TN, KS = kBK / 16;
  const int lane = threadIdx.x & 63, w = wave_id(), wm = w / C::WN, wn = w % C::WN;
  const int ktail = static_cast<int>((k1 - k0) % kBK);
  const Side<C::BM, TM, C::NW, KA, true> sa(a.a, wm, lane, w, ktail);
  const Side<C::BN, TN, C::NW, KB, false> sb(a.b, wn, lane, w, ktail);
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x16{};
  const int nkt = static_cast<int>((k1 - k0 + kBK - 1) / kBK);
  const int steps = SPLIT ? nkt * kPairs : nkt;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(smem));
  unsigned char* const bt = smem + 2 * C::LDS_A;
  int fpair = 0, fkt = 0;  // the k tile to fetch
  auto fetch_a = [&](int buf) __attribute__((always_inline)) {
    const int64_t pa = SPLIT ? (kPairA >> (2 * fpair)) & 3 : 0;
    sa.fetch(a.a, pa, m0, a.m, k0 + static_cast<int64_t>(fkt) * kBK, k1, lds0 + buf * C::LDS_A, w);
  };
  auto fetch_b = [&]() __attribute__((always_inline)) {
    const int64_t pb = SPLIT ? (kPairB >> (2 * fpair)) & 3 : 0;
    sb.fetch(a.b, pb, n0, a.n, k0 + static_cast<int64_t>(fkt) * kBK, k1, lds0 + 2 * C::LDS_A, w);
    if (++fkt == nkt) fkt = 0, ++fpair;
  };
  fetch_a(0);
  fetch_b();
  for (int st = 0; st < steps; ++st) {
    const bool more = st + 1 < steps;
    wait_vmcnt0();
    __syncthreads();  // every wave's loads of this tile are done; everyone has finished the tile before
    const unsigned char* at = smem + (st & 1) * C::LDS_A;
    u32x4 af[2][TM], bf[KS][TN];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int t = 0; t < TN; ++t) bf[ks][t] = sb.frag(bt, t, ks);
#pragma unroll
    for (int t = 0; t < TM; ++t) af[0][t] = sa.frag(at, t, 0);
    if (more) fetch_a((st + 1) & 1);
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): b's fragments are in registers
    __syncthreads();
    if (more) fetch_b();
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if (ks + 1 < KS) {
#pragma unroll
        for (int t = 0; t < TM; ++t) af[(ks + 1) & 1][t] = sa.frag(at, t, ks + 1);
      }
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = mfma32_dt<DT>(af[ks & 1][i], bf[ks][j], acc[i][j]);
      __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// One tile by k tiles that are C::NS deep in LDS: for tiles whose products take
// less than a load's latency. acc as above.
template <int DT, typename C, bool KA, bool KB, bool SPLIT>
__device__ __forceinline__ void deep_tile(const TileArgs& a, unsigned char* smem, f32x16 (&acc)[C::TM][C::TN], int m0,
                                          int n0, int64_t k0, int64_t k1) {
  constexpr int TM = C::TM, TN = C::TN, KS = kBK / 16, NS = C::NS, STAGE = C::LDS_A + C::LDS_B;
  const int lane = threadIdx.x & 63, w = wave_id(), wm = w / C::WN, wn = w % C::WN;
  const int ktail = static_cast<int>((k1 - k0) % kBK);
  const Side<C::BM, TM, C::NW, KA, true> sa(a.a, wm, lane, w, ktail);
  const Side<C::BN, TN, C::NW, KB, false> sb(a.b, wn, lane, w, ktail);
  constexpr int PER = decltype(sa)::BLOCKS + decltype(sb)::BLOCKS;
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x16{};
  const int nkt = static_cast<int>((k1 - k0 + kBK - 1) / kBK);
  const int steps = SPLIT ? nkt * kPairs : nkt;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(smem));
  int fpair = 0, fkt = 0, fbuf = 0, buf = 0;
  auto fetch = [&]() __attribute__((always_inline)) {
    const int64_t pa = SPLIT ? (kPairA >> (2 * fpair)) & 3 : 0, pb = SPLIT ? (kPairB >> (2 * fpair)) & 3 : 0;
    const int64_t kk = k0 + static_cast<int64_t>(fkt) * kBK;
    sa.fetch(a.a, pa, m0, a.m, kk, k1, lds0 + fbuf * STAGE, w);
    sb.fetch(a.b, pb, n0, a.n, kk, k1, lds0 + fbuf * STAGE + C::LDS_A, w);
    fbuf = fbuf + 1 == NS ? 0 : fbuf + 1;
    if (++fkt == nkt) fkt = 0, ++fpair;
  };
#pragma unroll
  for (int i = 0; i < NS - 1; ++i)
    if (i < steps) fetch();
  for (int st = 0; st < steps; ++st, buf = buf + 1 == NS ? 0 : buf + 1) {
    if (st + NS - 2 < steps)  // all but the NS - 2 later tiles' loads have landed
      __builtin_amdgcn_s_waitcnt(0x0f70 | (((NS - 2) * PER) & 15) | ((((NS - 2) * PER) >> 4) << 14));
    else
      wait_vmcnt0();
    __syncthreads();  // every wave's loads of this tile are done; everyone has finished the tile before
    if (st + NS - 1 < steps) fetch();
    const unsigned char* at = smem + buf * STAGE;
    u32x4 af[KS][TM], bf[KS][TN];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
      for (int t = 0; t < TM; ++t) af[ks][t] = sa.frag(at, t, ks);
#pragma unroll
      for (int t = 0; t < TN; ++t) bf[ks][t] = sb.frag(at + C::LDS_A, t, ks);
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = mfma32_dt<DT>(af[ks][i], bf[ks][j], acc[i][j]);
  }
}

// Stores a wave's 32 n rows (n tile j) of its 32 TM m columns, ES bytes each:
// every lane has a row's 16-column runs (`v`: as stored), which would make
// stores of 16 bytes in 64 places; through 8 KB of LDS of the wave's own (4 KB
// for 16-bit rows of 64) each instruction stores whole lines instead, the rows'
// 16-byte slots XOR-swizzled so that neither side meets a bank twice. `left`
// columns are inside the output, `rows` of the rows. add: fp32 only, to what is
// there. Every wave has left the tile loop.
template <int ES, int TM>
constexpr int put_rows_at_once() {
  return ES == 4 ? 16 : 32;
}
template <int ES, int TM>
constexpr int put_bytes() {
  return put_rows_at_once<ES, TM>() * TM * 32 * ES;
}
template <int ES, int TM>
__device__ __forceinline__ void put_rows(unsigned char* lds, const u32x4 (&v)[TM][ES], char* out, int64_t ld_b, int rows,
                                         int left, bool add) {
  constexpr int P = TM * 32 * ES, CH = P / 16, VE = 16 / ES, PASS = put_rows_at_once<ES, TM>();
  constexpr int SW = CH < 16 ? CH - 1 : 15;
  const int lane = threadIdx.x & 63, mine = lane & 31;
#pragma unroll
  for (int r0 = 0; r0 < 32; r0 += PASS) {
    __builtin_amdgcn_wave_barrier();  // the wave's own rows: LDS keeps its order, no workgroup barrier
    if (PASS == 32 || (mine >= r0 && mine < r0 + PASS)) {
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int q = 0; q < ES; ++q) {
          const int ch = (i * 32 + 16 * (lane >> 5)) * ES / 16 + q;
          *reinterpret_cast<u32x4*>(lds + (mine - r0) * P + ((ch ^ (mine & SW)) << 4)) = v[i][q];
        }
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int it = 0; it < PASS * CH / 64; ++it) {
      const int idx = it * 64 + lane, r = idx / CH, ch = idx % CH, row = r0 + r;
      const u32x4 w = *reinterpret_cast<const u32x4*>(lds + r * P + ((ch ^ (row & SW)) << 4));
      char* o = out + row * ld_b + ch * 16;
      if (row >= rows) continue;
      if ((ch + 1) * VE <= left) {
        if constexpr (ES == 4) {
          f32x4 x = __builtin_bit_cast(f32x4, w);
          if (add) x += *reinterpret_cast<const f32x4u*>(o);
          *reinterpret_cast<f32x4u*>(o) = x;
        } else {
          __builtin_nontemporal_store(__builtin_bit_cast(u32x4h, w), reinterpret_cast<u32x4h*>(o));
        }
      } else {
#pragma unroll
        for (int e = 0; e < VE - 1; ++e)
          if (ch * VE + e < left) {
            if constexpr (ES == 4) {
              float* f = reinterpret_cast<float*>(o) + e;
              *f = add ? *f + __uint_as_float(w[e]) : __uint_as_float(w[e]);
            } else {
              reinterpret_cast<uint16_t*>(o)[e] = static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1)));
            }
          }
      }
    }
  }
}

template <int DT>
__device__ __forceinline__ u32x4 pack8(const float* q) {
  u32x4 w;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    w[e] = DT == PDH_BF16 ? pack2<__hip_bfloat16>(q[2 * e], q[2 * e + 1]) : pack2<_Float16>(q[2 * e], q[2 * e + 1]);
  return w;
}

using Big = Config<2, 2, 4, 2, 0>;    // 256 x 128 tiles
using Small = Config<2, 2, 2, 1, 3>;  // 128 x 64: a quarter of one
// The gradient products of widths that would leave half a 256-feature tile empty.
using Half = Config<1, 4, 4, 2, 0>;      // 128 x 256
using Quarter = Config<1, 4, 2, 2, 0>;   // 64 x 256
static_assert(Small::LDS <= Big::LDS, "one kernel runs both");
static_assert(4 * put_bytes<2, 4>() <= Big::LDS_A && 4 * put_bytes<4, 4>() <= Big::LDS_A && 4 * put_bytes<2, 2>() <= Small::LDS &&
                  4 * put_bytes<4, 4>() <= Half::LDS && 4 * put_bytes<4, 2>() <= Quarter::LDS,
              "the stores' rows fit");
constexpr int kStrip = 128;        // vocabulary entries of a forward's strip

// The logits' tiles, [0, big) whole and the rest quartered (`small` of them),
// so that the last round of workgroups is a short one.
struct LogitTiles {
  TileArgs t;  // a: w (m: vocabulary), b: x (n: tokens)
  int big, small;
};
template <int DT, bool SPLIT, typename P, typename F>
__device__ __forceinline__ void logit_tile(const LogitTiles& l, unsigned char* smem, const P& p, const F& epilogue) {
  bool second;
  const int id = run_id(l.big, l.small, second);
  if (id < 0) return;
  const Tile t = tile_of(l.t, second ? l.big + id / 4 : id);
  int m0 = t.m * Big::BM, n0 = t.n * Big::BN;
  if (!second) {
    f32x16 acc[Big::TM][Big::TN];
    const auto info = epilogue.template info<Big>(p, n0);
    xent_tile<DT, Big, true, true, SPLIT>(l.t, smem, acc, m0, n0, 0, l.t.k);
    epilogue.template store<Big>(p, acc, info, m0, n0, smem);
  } else {
    m0 += (id & 1) * Small::BM, n0 += ((id >> 1) & 1) * Small::BN;
    if (m0 >= l.t.m || n0 >= l.t.n) return;
    f32x16 acc[Small::TM][Small::TN];
    const auto info = epilogue.template info<Small>(p, n0);
    deep_tile<DT, Small, true, true, SPLIT>(l.t, smem, acc, m0, n0, 0, l.t.k);
    epilogue.template store<Small>(p, acc, info, m0, n0, smem);
  }
}

// ---------------------------------------------------------------- forward

struct FwdArgs {
  LogitTiles l;
  const int64_t* targets;
  float2* part;  // [strips][tokens]: (max, sum of exp(z - max)) of kStrip vocabulary entries
  float* zt;     // [tokens]: the target's logit
};

// Joins (m, s) and (om, os), sums of exponentials below their maxima.
__device__ __forceinline__ void join(float& m, float& s, float om, float os) {
  const float mn = nan_max(m, om);
  const float b = mn == -__builtin_inff() ? 0.f : mn;  // nothing but -inf so far sums to 0, not NaN
  s = s * fast_exp2((m - b) * kLog2e) + os * fast_exp2((om - b) * kLog2e);
  m = mn;
}

// What the epilogue needs of a lane's tokens, read before the products.
template <int TN>
struct FwdInfo {
  int target[TN];  // -1: none
};

struct FwdEpilogue {
  template <typename C>
  __device__ __forceinline__ FwdInfo<C::TN> info(const FwdArgs& p, int n0) const {
    FwdInfo<C::TN> f;
#pragma unroll
    for (int j = 0; j < C::TN; ++j) {
      const int n = n0 + 32 * ((wave_id() % C::WN) * C::TN + j) + (threadIdx.x & 31);
      const int64_t t = n < p.l.t.n ? p.targets[n] : -1;
      f.target[j] = t >= 0 && t < p.l.t.m ? static_cast<int>(t) : -1;
    }
    return f;
  }
  template <typename C>
  __device__ __forceinline__ void store(const FwdArgs& p, f32x16 (&acc)[C::TM][C::TN], const FwdInfo<C::TN>& f, int m0,
                                        int n0, unsigned char* lds) const {
    constexpr int TM = C::TM, TN = C::TN;
    const int lane = threadIdx.x & 63, w = wave_id(), wm = w / C::WN, wn = w % C::WN, g = lane >> 5;
    const int vocab = p.l.t.m, tokens = p.l.t.n;
    const int vw = m0 + 32 * wm * TM, v0 = vw + 16 * g;  // the wave's entries, the lane's first
    float mxs[TN], sums[TN], zs[TN];
    bool hit[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      if (vw + 32 * TM > vocab) {  // entries past the vocabulary weigh nothing
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (v0 + 32 * i + e >= vocab) acc[i][j][e] = -__builtin_inff();
      }
      float mx = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, acc[i][j][e]);
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float base = mx == -__builtin_inff() ? 0.f : mx * kLog2e;
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) s += fast_exp2(__builtin_fmaf(acc[i][j][e], kLog2e, -base));
      s += __shfl_xor(s, 32, 64);
      mxs[j] = mx, sums[j] = s;
      const int tl = f.target[j] - v0;
      hit[j] = f.target[j] >= 0 && tl >= 0 && tl < 32 * TM && (tl & 16) == 0;
      zs[j] = 0.f;
      if (hit[j]) {  // this lane holds the target's logit
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (tl == 32 * i + e) zs[j] = acc[i][j][e];
      }
    }
    if constexpr (32 * TM < kStrip) {  // the strip's two waves meet in LDS
      static_assert(64 * TM == kStrip && C::WM == 2, "two waves a strip");
      __syncthreads();  // the tile loop's last reads are over
      float2* sh = reinterpret_cast<float2*>(lds);
      if (wm == 1 && g == 0)
#pragma unroll
        for (int j = 0; j < TN; ++j) sh[(wn * TN + j) * 32 + lane] = make_float2(mxs[j], sums[j]);
      __syncthreads();
      if (wm == 0) {
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const float2 o = sh[(wn * TN + j) * 32 + (lane & 31)];
          join(mxs[j], sums[j], o.x, o.y);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = n0 + 32 * (wn * TN + j) + (lane & 31);
      if (n < tokens && g == 0 && vw < vocab && (32 * TM == kStrip || wm == 0))
        p.part[static_cast<int64_t>(vw / kStrip) * tokens + n] = make_float2(mxs[j], sums[j]);
      if (hit[j]) p.zt[n] = zs[j];
    }
  }
};

template <int DT, bool SPLIT>
__global__ __launch_bounds__(256, 2) void xent_fwd(FwdArgs p) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[Big::LDS];
  logit_tile<DT, SPLIT>(p.l, smem, p, FwdEpilogue{});
}

// Joins the strips of 16 tokens, 64 lanes a token with eight loads in flight
// each: lse and loss (8192 tokens, 393 strips: 8 us; 32 lanes a token and a
// load at a time, 13).
__global__ __launch_bounds__(1024) void xent_join(const float2* __restrict__ part, const float* __restrict__ zt,
                                                  const int64_t* __restrict__ targets, int strips, int64_t n_tokens,
                                                  int64_t vocab, int64_t ignore, float* __restrict__ loss,
                                                  float* __restrict__ lse, int* __restrict__ bad) {
  __shared__ float2 sh[64][16];
  const int tok = threadIdx.x & 15, q = threadIdx.x >> 4;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * 16 + tok;
  float m = -__builtin_inff(), s = 0.f;
  if (n < n_tokens) {
    for (int i0 = q; i0 < strips; i0 += 512) {
      float2 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        v[u] = i0 + 64 * u < strips ? part[static_cast<int64_t>(i0 + 64 * u) * n_tokens + n]
                                    : make_float2(-__builtin_inff(), 0.f);
#pragma unroll
      for (int u = 0; u < 8; ++u) join(m, s, v[u].x, v[u].y);
    }
  }
  sh[q][tok] = make_float2(m, s);
  __syncthreads();
  if (q < 8) {
    for (int i = q + 8; i < 64; i += 8) join(m, s, sh[i][tok].x, sh[i][tok].y);
  }
  __syncthreads();
  if (q < 8) sh[q][tok] = make_float2(m, s);
  __syncthreads();
  if (q == 0 && n < n_tokens) {
    for (int i = 1; i < 8; ++i) join(m, s, sh[i][tok].x, sh[i][tok].y);
    const float l = m + logf(s);
    const int64_t t = targets[n];
    const bool live = t >= 0 && t < vocab && t != ignore;
    lse[n] = l;
    loss[n] = live ? l - zt[n] : 0.f;
    if (!live && t != ignore && bad) atomicAdd(bad, 1);
  }
}

// --------------------------------------------------------------- backward

struct GradArgs {
  LogitTiles l;        // a: w from the piece's first row (m: its entries)
  const int64_t* targets;
  const float* lse;
  const float* dloss;
  const float* most;   // dz is taken over it,
  float raise;         // times this power of two
  uint16_t* dz;        // [planes][tokens][ldz]
  int64_t ldz, plane;  // elements
  int64_t v0;          // the piece's first vocabulary entry
  int64_t vocab, ignore;
};

constexpr int kNoToken = INT32_MIN;
template <int TN>
struct DzInfo {
  int target[TN];  // from the piece's first entry; kNoToken: an ignored token
  float g[TN], lse2[TN];
};

template <int DT, bool SPLIT>
struct DzEpilogue {
  template <typename C>
  __device__ __forceinline__ DzInfo<C::TN> info(const GradArgs& p, int n0) const {
    DzInfo<C::TN> f;
#pragma unroll
    for (int j = 0; j < C::TN; ++j) {
      const int n = n0 + 32 * ((wave_id() % C::WN) * C::TN + j) + (threadIdx.x & 31);
      const int64_t t = n < p.l.t.n ? p.targets[n] : -1;
      const bool live = t >= 0 && t < p.vocab && t != p.ignore;
      f.target[j] = live ? static_cast<int>(t - p.v0) : kNoToken;
      f.g[j] = live ? p.dloss[n] / *p.most * p.raise : 0.f;
      // an ignored token's x is zeros: exp2(-inf) times 0 (but for an entry of w that is not finite: below)
      f.lse2[j] = live ? p.lse[n] * kLog2e : __builtin_inff();
    }
    return f;
  }
  template <typename C>
  __device__ __forceinline__ void store(const GradArgs& p, f32x16 (&acc)[C::TM][C::TN], const DzInfo<C::TN>& f, int m0,
                                        int n0, unsigned char* lds) const {
    constexpr int TM = C::TM, TN = C::TN;
    const int lane = threadIdx.x & 63, w = wave_id(), wm = w / C::WN, wn = w % C::WN, g = lane >> 5;
    const int cw = m0 + 32 * wm * TM;  // the wave's first column of dz
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const bool live = f.target[j] != kNoToken;
      const int tl = live ? f.target[j] - (cw + 16 * g) : -1;
#pragma unroll
      for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = fast_exp2(__builtin_fmaf(acc[i][j][e], kLog2e, -f.lse2[j]));
        const int at = tl - 32 * i;
        if (at >= 0 && at < 16) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (at == e) acc[i][j][e] -= 1.f;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] *= f.g[j];
      }
    }
    if (cw + 32 * TM > p.l.t.m) {  // entries past the vocabulary are zero
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (cw + 32 * i + 16 * g + e >= p.l.t.m) acc[i][j][e] = 0.f;
    }
    __syncthreads();  // the tile loop's last reads are over: LDS serves the stores
    lds += w * put_bytes<2, TM>();
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int nw = n0 + 32 * (wn * TN + j);
#pragma unroll
      for (int pl = 0; pl < (SPLIT ? 3 : 1); ++pl) {
        u32x4 v[TM][2];
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = acc[i][j][8 * q + e];
            v[i][q] = pack8<DT>(x);
            if constexpr (SPLIT) {  // what this term leaves (exact)
#pragma unroll
              for (int e = 0; e < 8; ++e)
                acc[i][j][8 * q + e] -= __uint_as_float(e & 1 ? v[i][q][e >> 1] & 0xffff0000u : v[i][q][e >> 1] << 16);
            }
          }
        // an ignored token's dz is zero whatever w holds, as stored: half the selects of one an element, and
        // none where all 32 tokens are live (a token in 20 ignored, without / with: backward 8192 x 768 x 50257
        // bf16 1905 / 1910 us, 4096 x 4096 4398 / 4412, 16384 x 64 x 20000 432 / 438)
        if (__any(f.target[j] == kNoToken)) {
#pragma unroll
          for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
              for (int e = 0; e < 4; ++e) v[i][q][e] = f.target[j] == kNoToken ? 0u : v[i][q][e];
        }
        put_rows<2, TM>(lds, v, reinterpret_cast<char*>(p.dz + pl * p.plane + static_cast<int64_t>(nw) * p.ldz + cw),
                        p.ldz * 2, p.l.t.n - nw, static_cast<int>(p.ldz) - cw, false);
      }
    }
  }
};

template <int DT, bool SPLIT>
__global__ __launch_bounds__(256, 2) void xent_dz(GradArgs p) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[Big::LDS];
  logit_tile<DT, SPLIT>(p.l, smem, p, DzEpilogue<DT, SPLIT>{});
}

// The gradient products, both in one launch so that their tiles fill the chip
// together: a: x or w with its features contiguous (m: features), b: dz, by its
// columns (dw: n vocabulary, k tokens) or rows (dx: n tokens, k vocabulary).
struct ProdArgs {
  TileArgs w, x;
  int tiles_w, tiles_x;  // with slices
  int x_first;           // the longer tiles go first
  void* dw;              // or its parts, [slices][vocabulary][ldp] (w.slices > 1)
  float* parts;          // dx's, [slices][tokens][ldp]
  int64_t lddw, ldp, slice_w, slice;
  const float* most;     // dw is times it,
  float down;            // and this
  int add;               // dx's parts of an earlier piece are there
};

template <int DT, int ODT, typename C, bool KB, bool SPLIT>
__device__ __forceinline__ void prod_tile(const TileArgs& a, int id, unsigned char* smem, char* out, int64_t ld,
                                          int64_t slice, float sc, bool add) {
  constexpr int TM = C::TM, TN = C::TN, ES = ODT == PDH_F32 ? 4 : 2;
  const Tile t = tile_of(a, id);
  const int m0 = t.m * C::BM, n0 = t.n * C::BN;
  const int w = wave_id(), wm = w / C::WN, wn = w % C::WN;
  f32x16 acc[TM][TN];
  const int64_t k0 = static_cast<int64_t>(t.slice) * a.kslice, k1 = k0 + a.kslice < a.k ? k0 + a.kslice : a.k;
  xent_tile<DT, C, false, KB, SPLIT>(a, smem, acc, m0, n0, k0, k1);
  __syncthreads();  // the tile loop's last reads are over: LDS serves the stores
  unsigned char* lds = smem + w * put_bytes<ES, TM>();
  const int cw = m0 + 32 * wm * TM;
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int nw = n0 + 32 * (wn * TN + j);
    u32x4 v[TM][ES];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int q = 0; q < ES; ++q) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 16 / ES; ++e) x[e] = acc[i][j][16 / ES * q + e] * sc;
        if constexpr (ES == 4)
          v[i][q] = u32x4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
        else
          v[i][q] = pack8<ODT>(x);
      }
    put_rows<ES, TM>(lds, v, out + (t.slice * slice + static_cast<int64_t>(nw) * ld + cw) * ES, ld * ES, a.n - nw,
                     a.m - cw, add);
  }
}

template <int DT, int ODT, typename C, bool SPLIT>
__global__ __launch_bounds__(256, 2) void xent_prod(ProdArgs p) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[C::LDS];
  bool second;
  const int id = run_id(p.x_first ? p.tiles_x : p.tiles_w, p.x_first ? p.tiles_w : p.tiles_x, second);
  if (id < 0) return;
  if (second != static_cast<bool>(p.x_first))
    prod_tile<DT, PDH_F32, C, true, SPLIT>(p.x, id, smem, reinterpret_cast<char*>(p.parts), p.ldp, p.slice, 1.f, p.add);
  else if (p.w.slices > 1)
    prod_tile<DT, PDH_F32, C, false, SPLIT>(p.w, id, smem, static_cast<char*>(p.dw), p.ldp, p.slice_w, 1.f, false);
  else
    prod_tile<DT, ODT, C, false, SPLIT>(p.w, id, smem, static_cast<char*>(p.dw), p.lddw, 0, *p.most * p.down, false);
}

// A gradient = *most * down * the sum of its parts, in order. A row without a
// target (dx: `targets` given) is zero, whatever w made of its zeros.
template <int DT>
__global__ __launch_bounds__(256) void xent_sum(const float* __restrict__ part, void* dx, int64_t rows, int d,
                                               int64_t ld, int64_t slice, int slices, const float* __restrict__ most,
                                               float down, const int64_t* __restrict__ targets, int64_t vocab,
                                               int64_t ignore) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t per = ld / 4, n = i / per;
  const int c = static_cast<int>(i - n * per) * 4;
  if (n >= rows || c >= d) return;
  const float* p = part + n * ld + c;
  f32x4 s{};
  for (int q0 = 0; q0 < slices; q0 += 8) {  // eight loads in flight, added in order
    f32x4 v[8];
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (q0 + q < slices) v[q] = *reinterpret_cast<const f32x4*>(p + (q0 + q) * slice);
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (q0 + q < slices) s += v[q];
  }
  s *= *most * down;
  if (targets) {
    const int64_t t = targets[n];
    if (t < 0 || t >= vocab || t == ignore) s = f32x4{};
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (c + e < d) st_dt<DT>(dx, n * d + c + e, s[e]);
}

// *most = the largest finite |dloss| of a live token, 1 where there is none:
// dz is taken over it. (Over an infinite one, or over 1 beside it, fp16's dz of
// every other token would leave its range.) One workgroup, sixteen tokens' loads
// in flight a lane (8192 tokens: 7 us; one at a time, 36).
struct MostArgs {
  const float* dloss;  // NULL: none to do
  const int64_t* targets;
  int64_t n, vocab, ignore;
  float* most;
};
__device__ __forceinline__ void most_dloss(const MostArgs& p) {
  __shared__ float sh[4];
  constexpr int U = 16;
  float mx = 0.f;
  for (int64_t i0 = threadIdx.x; i0 < p.n; i0 += 256 * U) {
    int64_t t[U];
    float d[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = i0 + 256 * u < p.n ? i0 + 256 * u : i0;
      t[u] = p.targets[i];
      d[u] = p.dloss[i];
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (t[u] >= 0 && t[u] < p.vocab && t[u] != p.ignore && fabsf(d[u]) < __builtin_inff()) mx = fmaxf(mx, fabsf(d[u]));
  }
  mx = wave_max(mx);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3]));
  if (threadIdx.x == 0) *p.most = mx > 0.f ? mx : 1.f;
}

// An operand made fit for the direct loads: rows of `dp` (a multiple of 8)
// 16-bit values, zero past d. fp32 rows become three planes of bf16 terms,
// 16-bit ones of odd width, stride or alignment a padded copy. The backward's
// tokens are always copied: an ignored one's row comes out zero, so that what a
// padded batch holds there (infinities, NaN) never meets dw's products (8192 x
// 768 x 50257 bf16 1931 us either way, 4096 x 4096 x 50257 4394 -> 4423).
struct PackArgs {
  const void* src;  // NULL: read in place
  int64_t ld, rows;
  int d, dp;
  uint16_t* dst;
  int64_t plane;
  const int64_t* targets;  // NULL: every row; or a row without a target in [0, vocab) is zero
  int64_t vocab, ignore;
};
template <int DT>
__device__ __forceinline__ void pack_rows(const PackArgs& p, int64_t i) {
  const int64_t per = p.dp / 8, n = i / per;
  const int c = static_cast<int>(i - n * per) * 8;
  if (n >= p.rows) return;
  uint16_t* o = p.dst + n * p.dp + c;
  if (p.targets) {
    const int64_t t = p.targets[n];
    if (t < 0 || t >= p.vocab || t == p.ignore) {
#pragma unroll
      for (int pl = 0; pl < (DT == PDH_F32 ? 3 : 1); ++pl) *reinterpret_cast<u32x4*>(o + pl * p.plane) = u32x4{};
      return;
    }
  }
  if constexpr (DT == PDH_F32) {
    const float* x = static_cast<const float*>(p.src) + n * p.ld + c;
    float v[8];
    if (c + 8 <= p.d) {
      const f32x4u a = reinterpret_cast<const f32x4u*>(x)[0], b = reinterpret_cast<const f32x4u*>(x)[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = c + e < p.d ? x[e] : 0.f;
    }
#pragma unroll
    for (int pl = 0; pl < 3; ++pl) {
      u32x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        w[e] = pack2<__hip_bfloat16>(v[2 * e], v[2 * e + 1]);
        v[2 * e] -= __uint_as_float(w[e] << 16);
        v[2 * e + 1] -= __uint_as_float(w[e] & 0xffff0000u);
      }
      *reinterpret_cast<u32x4*>(o + pl * p.plane) = w;
    }
  } else {
    const uint16_t* x = static_cast<const uint16_t*>(p.src) + n * p.ld + c;
    u32x4 w{};
    if (c + 8 <= p.d) {
      w = *reinterpret_cast<const u32x4h*>(x);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < p.d) w[e >> 1] |= static_cast<uint32_t>(x[e]) << (16 * (e & 1));
    }
    *reinterpret_cast<u32x4*>(o) = w;
  }
}

// What the products wait for, in one launch: w's and x's workgroups, then dloss's largest value in one more.
struct PrepArgs {
  PackArgs w, x;
  MostArgs most;
  uint32_t blocks_w, blocks_x;
};
template <int DT>
__global__ __launch_bounds__(256) void xent_prep(PrepArgs p) {
  const uint32_t b = blockIdx.x;
  if (b < p.blocks_w)
    pack_rows<DT>(p.w, static_cast<int64_t>(b) * 256 + threadIdx.x);
  else if (b < p.blocks_w + p.blocks_x)
    pack_rows<DT>(p.x, static_cast<int64_t>(b - p.blocks_w) * 256 + threadIdx.x);
  else
    most_dloss(p.most);
}

// ------------------------------------------------------------------- host

// dz of one piece of the vocabulary (backward 8192 x 768 x 50257 bf16, one
// piece of 823 MB: pieces of 512 MiB take 0.7% longer, of 256 or 128 MiB 5%), and
// a gradient's parts
constexpr int64_t kPieceBytes = int64_t{1} << 30, kPartBytes = int64_t{1} << 31;

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

struct Problem {
  int64_t n, d, v;  // tokens, width, vocabulary
  int64_t ldx, ldw;
  const void* x;
  const void* w;
  int dtype;
  int planes() const { return dtype == PDH_F32 ? 3 : 1; }
  int64_t dp() const { return up(d, 8); }
  // read in place: 16-bit rows of whole 16-byte chunks, 256 of them within the loads' reach
  static bool fit(const void* p, int64_t ld, int64_t d, int dtype) {
    return dtype != PDH_F32 && d % 8 == 0 && ld % 8 == 0 && ld >= d && aligned16(p) && ld <= (int64_t{1} << 21);
  }
};

// A bump allocator over the caller's workspace; without one it measures.
struct Space {
  char* base;
  size_t used = 0;
  void* take(int64_t bytes) {
    const size_t at = used;
    used += static_cast<size_t>(up(bytes, 1024));
    return base ? base + at : nullptr;
  }
};

unsigned blocks_for(int64_t threads) { return static_cast<unsigned>((threads + 255) / 256); }

// The operand of rows p[rows][d]: in place, or in ws, where `pack` says how it comes there.
Operand place(const void* p, int64_t ld, int64_t rows, const Problem& q, Space& ws, bool in_place, PackArgs& pack) {
  pack = PackArgs{};
  if (in_place) return Operand{static_cast<const char*>(p), ld * 2, 0};
  const int64_t dp = q.dp(), plane = rows * dp;
  auto* dst = static_cast<uint16_t*>(ws.take(plane * 2 * q.planes()));
  pack = PackArgs{p, ld, rows, static_cast<int>(q.d), static_cast<int>(dp), dst, plane, nullptr, 0, 0};
  return Operand{reinterpret_cast<const char*>(dst), dp * 2, plane * 2};
}

// Launches what there is to prepare.
int prepare(const char* fn, const Problem& q, PackArgs w, PackArgs x, const MostArgs& most, hipStream_t s) {
  PrepArgs p{w, x, most, 0, 0};
  if (w.src) p.blocks_w = blocks_for(w.rows * (w.dp / 8));
  if (x.src) p.blocks_x = blocks_for(x.rows * (x.dp / 8));
  const unsigned blocks = p.blocks_w + p.blocks_x + (most.dloss ? 1 : 0);
  if (blocks == 0) return PDH_OK;
  if (q.dtype == PDH_F32)
    xent_prep<PDH_F32><<<dim3(blocks), 256, 0, s>>>(p);
  else
    xent_prep<PDH_BF16><<<dim3(blocks), 256, 0, s>>>(p);  // 16-bit rows are copied as they are
  return check_launch(fn);
}

template <typename C>
TileArgs tiles(Operand a, Operand b, int64_t m, int64_t n, int64_t k, int64_t kslice) {
  TileArgs t{};
  t.a = a, t.b = b;
  t.m = static_cast<int>(m), t.n = static_cast<int>(n), t.k = static_cast<int>(k);
  t.tiles_m = static_cast<int>((m + C::BM - 1) / C::BM);
  t.tiles_n = static_cast<int>((n + C::BN - 1) / C::BN);
  t.kslice = static_cast<int>(kslice);
  t.slices = static_cast<int>((k + kslice - 1) / kslice);
  t.group = t.tiles_n < 8 ? t.tiles_n : 8;
  return t;
}
int64_t count(const TileArgs& t) { return static_cast<int64_t>(t.tiles_m) * t.tiles_n * t.slices; }

// Workgroups of these kernels that run at a time on the current device, on which
// the plan, and so the workspace and the order of the sums, depends.
int64_t slots() {
  static thread_local int of = -1, cus = 0;
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess) dev = -1;
  if (dev != of || !cus) of = dev, cus = pdh_device_cus();
  return 2 * (cus ? cus : 256);
}

// The logits' tiles past the last whole round run as quarters where those take less time: a
// quarter takes 0.33 of a tile's time.
LogitTiles logit_tiles(const TileArgs& t) {
  const int64_t all = count(t), s = slots(), left = all % s;
  const bool quarter = left > 0 && 0.33 * static_cast<double>((4 * left + s - 1) / s) < 1.0;
  const int64_t big = quarter ? all - left : all;
  return LogitTiles{t, static_cast<int>(big), static_cast<int>(quarter ? 4 * left : 0)};
}

// The time at which `s` slots end n1 jobs of d1 and then n2 of d2 <= d1, each
// slot taking the next job when it is free.
double makespan(int64_t n1, double d1, int64_t n2, double d2, int64_t s) {
  const int64_t q = n1 / s, r = n1 % s;  // r slots are free at (q + 1) d1, the rest at q d1
  const double early = q * d1, late = early + (r ? d1 : 0.0);
  if (n2 == 0) return r ? late : early;
  double best = 1e300;
  for (int64_t i = 1; best == 1e300; ++i) {
    for (const double t : {early + i * d2, late + i * d2}) {
      const int64_t fit = (s - r) * static_cast<int64_t>((t - early) / d2 + 1e-9) +
                          r * std::max<int64_t>(0, static_cast<int64_t>((t - late) / d2 + 1e-9));
      if (t >= late && fit >= n2) best = std::min(best, t);
    }
  }
  return best;
}

// The gradient products' tiles: 256 features where the width fills them, 128
// where half of the last one would be empty, 64 for widths up to that.
// Backward at 16384 tokens x 20000 entries, us, always 256 and dw in one part /
// the choice and dw's parts below: bf16 width 64 574 / 448, 128 627 / 522 (and
// 256, with parts alone, 739 / 677), 640 1478 / 1402; fp32 width 32 4040 / 1817.
enum class Prod { kBig, kHalf, kQuarter };
Prod pick_prod(int64_t d) { return d <= 64 ? Prod::kQuarter : (d + 127) / 128 % 2 ? Prod::kHalf : Prod::kBig; }

// k columns of a slice, and slices, of the two gradient products of the first
// piece: the parts that are summed are those that its launch writes (a later
// piece, no longer, adds to them).
struct Slices {
  int64_t kw, w, kx, x;
};

// Those that end both products soonest, in k tiles' time: a tile's own cost is
// its k tiles and about 5 for its start and stores, a slice's the traffic of its
// part, added and read again (9e-7 k tiles an element at 4.5 TB/s, 2 us a k
// tile); dw's parts are one more launch, and there are some only where its tiles
// leave compute units without one. Backward with dw in one part / in those, us:
// 16000 x 700 x 1500 fp16 340 / 187, 30000 x 1100 x 1000 bf16 657 / 337,
// 5000 x 4096 x 300 bf16 157 / 116, 4000 x 384 x 6000 fp32 608 / 402.
Slices pick_slices(const Problem& q, int64_t piece) {
  const Prod kind = pick_prod(q.d);
  const int64_t bm = kind == Prod::kBig ? Big::BM : kind == Prod::kHalf ? Half::BM : Quarter::BM;
  const int64_t bn = kind == Prod::kBig ? Big::BN : Half::BN, mt = (q.d + bm - 1) / bm, dp = q.dp();
  const int64_t tw = mt * ((piece + bn - 1) / bn), tx = mt * ((q.n + bn - 1) / bn), free = slots();
  const double terms = (q.dtype == PDH_F32 ? kPairs : 1) * (kind == Prod::kQuarter ? 0.6 : 1.0);
  static constexpr int kTry[] = {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16, 20, 24, 28, 32, 40, 48, 56, 64};
  const int64_t most_w = tw < free ? std::min<int64_t>(q.n / 512, kPartBytes / (piece * dp * 4)) : 1;
  const int64_t most_x = std::min<int64_t>(piece / 256, kPartBytes / (q.n * dp * 4));
  double best = 1e300;
  int64_t bw = 1, bx = 1;
  for (const int64_t w : kTry) {
    if (w > 1 && w > most_w) break;
    const double dw = terms * ((q.n + w * kBK - 1) / (w * kBK)) + 5;
    const double cost_w = w > 1 ? 9e-7 * w * piece * dp + 2.5 : 0;
    for (const int64_t x : kTry) {
      if (x > 1 && x > most_x) break;
      const double dx = terms * ((piece + x * kBK - 1) / (x * kBK)) + 5;
      const double t = cost_w + 9e-7 * x * q.n * dp + (dx > dw ? makespan(tx * x, dx, tw * w, dw, free)
                                                               : makespan(tw * w, dw, tx * x, dx, free));
      if (t < best) best = t, bw = w, bx = x;
    }
  }
  Slices r;
  r.kw = up((q.n + bw - 1) / bw, kBK), r.w = (q.n + r.kw - 1) / r.kw;
  // a piece of the whole vocabulary is rounded up to tiles, past which no slice may lie
  const int64_t first = std::min(piece, q.v);
  r.kx = up((piece + bx - 1) / bx, kBK), r.x = (first + r.kx - 1) / r.kx;
  return r;
}

int check(const char* fn, int64_t n, int64_t d, int64_t v, int64_t ldx, int64_t ldw, int dtype) {
  PDH_REQUIRE(dtype == PDH_F32 || dtype == PDH_BF16 || dtype == PDH_F16, PDH_EUNSUPPORTED, "%s: dtype %d", fn, dtype);
  PDH_REQUIRE(n >= 0 && d >= 1 && v >= 1, PDH_EINVAL, "%s: need tokens >= 0, width >= 1, vocabulary >= 1 (got %lld, %lld, %lld)",
              fn, (long long)n, (long long)d, (long long)v);
  PDH_REQUIRE(n <= (int64_t{1} << 24) && v <= (int64_t{1} << 24) && d <= (int64_t{1} << 18), PDH_EUNSUPPORTED,
              "%s: at most 2^24 tokens and vocabulary entries and 2^18 features", fn);
  // every launch stays under 2^32 threads (packing: one for 8 elements of x and of w)
  PDH_REQUIRE(n * v <= (int64_t{1} << 38) && std::max(n, v) * up(d, 8) <= (int64_t{1} << 33), PDH_EUNSUPPORTED,
              "%s: at most 2^38 logits and 2^33 elements of x or w in a call", fn);
  PDH_REQUIRE(ldx >= 0 && ldw >= 0, PDH_EINVAL, "%s: row strides must be >= 0", fn);
  return PDH_OK;
}

// The forward's workspace (base NULL: measured) and its operands' places. Plans
// touch no memory: the caller checks what they used before it launches.
struct FwdPlan {
  Operand w, x;
  PackArgs pack_w, pack_x;
  TileArgs t;
  float2* part;
  float* zt;
  int strips;
};
FwdPlan plan_fwd(const Problem& q, Space& ws, bool fit_x, bool fit_w) {
  FwdPlan p{};
  p.w = place(q.w, q.ldw, q.v, q, ws, fit_w, p.pack_w);
  p.x = place(q.x, q.ldx, q.n, q, ws, fit_x, p.pack_x);
  p.t = tiles<Big>(p.w, p.x, q.v, q.n, q.dp(), up(q.dp(), kBK));
  p.strips = static_cast<int>((q.v + kStrip - 1) / kStrip);
  p.part = static_cast<float2*>(ws.take(static_cast<int64_t>(p.strips) * q.n * 8));
  p.zt = static_cast<float*>(ws.take(q.n * 4));
  return p;
}

struct BwdPlan {
  Operand w, x;
  PackArgs pack_w, pack_x;
  uint16_t* dz;
  float* parts;
  float* most;
  float* parts_w;  // dw's parts of a piece, where there are any
  int64_t piece;   // vocabulary entries of a piece (the last one's may be fewer)
  Slices slices;
};
BwdPlan plan_bwd(const Problem& q, Space& ws, bool fit_w) {
  BwdPlan p{};
  p.w = place(q.w, q.ldw, q.v, q, ws, fit_w, p.pack_w);
  p.x = place(q.x, q.ldx, q.n, q, ws, false, p.pack_x);
  const int64_t all = up(q.v, 256), most = kPieceBytes / (q.n * 2 * q.planes()) / 256 * 256;
  // (2^22 entries keep a tile's rows of dz within the loads' 32-bit offsets: that many only of 128 tokens or fewer)
  p.piece = std::min(std::min(all, int64_t{1} << 22), std::max<int64_t>(most, 256));
  p.dz = static_cast<uint16_t*>(ws.take(q.n * p.piece * 2 * q.planes()));
  p.slices = pick_slices(q, p.piece);
  p.parts = static_cast<float*>(ws.take(p.slices.x * q.n * q.dp() * 4));
  if (p.slices.w > 1) p.parts_w = static_cast<float*>(ws.take(p.slices.w * p.piece * q.dp() * 4));
  p.most = static_cast<float*>(ws.take(4));
  return p;
}

template <int DT, bool SPLIT>
int run_fwd(const Problem& q, const FwdPlan& p, const int64_t* targets, int64_t ignore, float* loss, float* lse, int* bad,
            hipStream_t s) {
  if (int rc = prepare("pdh_linear_xent_fwd (pack)", q, p.pack_w, p.pack_x, MostArgs{}, s); rc != PDH_OK) return rc;
  const LogitTiles l = logit_tiles(p.t);
  xent_fwd<DT, SPLIT><<<run_grid(l.big, l.small), 256, 0, s>>>(FwdArgs{l, targets, p.part, p.zt});
  if (int rc = check_launch("pdh_linear_xent_fwd"); rc != PDH_OK) return rc;
  xent_join<<<dim3(static_cast<unsigned>((q.n + 15) / 16)), 1024, 0, s>>>(p.part, p.zt, targets, p.strips, q.n, q.v, ignore,
                                                                       loss, lse, bad);
  return check_launch("pdh_linear_xent_fwd (join)");
}

// Both gradient products of a piece: entries v0 .. v0 + nv - 1.
template <int DT, int ODT, typename C, bool SPLIT>
void run_prod(const Problem& q, const BwdPlan& p, const Operand& wv, const Operand& dz, int64_t v0, int64_t nv,
              float down, void* dw, hipStream_t s) {
  const int64_t dp = q.dp();
  void* rows = static_cast<char*>(dw) + v0 * q.d * (ODT == PDH_F32 ? 4 : 2);
  const bool split = p.slices.w > 1;
  ProdArgs a{};
  a.w = tiles<C>(p.x, dz, q.d, nv, q.n, p.slices.kw);
  a.x = tiles<C>(wv, dz, q.d, q.n, nv, p.slices.kx);
  a.tiles_w = static_cast<int>(count(a.w)), a.tiles_x = static_cast<int>(count(a.x));
  a.x_first = p.slices.kx > p.slices.kw;
  a.dw = split ? p.parts_w : rows;
  a.parts = p.parts, a.lddw = q.d, a.ldp = dp, a.slice_w = nv * dp, a.slice = q.n * dp;
  a.most = p.most, a.down = down, a.add = v0 > 0;
  xent_prod<DT, ODT, C, SPLIT><<<run_grid(a.tiles_w, a.tiles_x), 256, 0, s>>>(a);
  if (split)
    xent_sum<ODT><<<dim3(blocks_for(nv * (dp / 4))), 256, 0, s>>>(p.parts_w, rows, nv, static_cast<int>(q.d), dp,
                                                                 nv * dp, static_cast<int>(p.slices.w), p.most, down,
                                                                 nullptr, 0, 0);
}

template <int DT, int ODT, bool SPLIT>
int run_bwd(const Problem& q, const BwdPlan& p, const int64_t* targets, const float* lse, const float* dloss,
            int64_t ignore, void* dx, void* dw, hipStream_t s) {
  const MostArgs most{dloss, targets, q.n, q.v, ignore, p.most};
  const float raise = DT == PDH_F16 ? 16384.f : 1.f;
  PackArgs live = p.pack_x;
  live.targets = targets, live.vocab = q.v, live.ignore = ignore;
  if (int rc = prepare("pdh_linear_xent_bwd (pack)", q, p.pack_w, live, most, s); rc != PDH_OK) return rc;
  const int64_t dp = q.dp();
  for (int64_t v0 = 0; v0 < q.v; v0 += p.piece) {
    const int64_t nv = std::min(p.piece, q.v - v0), ldz = up(nv, 256);
    const Operand wv{p.w.p + v0 * p.w.pitch, p.w.pitch, p.w.plane};
    const Operand dz{reinterpret_cast<const char*>(p.dz), ldz * 2, q.n * ldz * 2};
    const GradArgs ga{logit_tiles(tiles<Big>(wv, p.x, nv, q.n, dp, up(dp, kBK))), targets, lse, dloss, p.most, raise,
                      p.dz, ldz, q.n * ldz, v0, q.v, ignore};
    xent_dz<DT, SPLIT><<<run_grid(ga.l.big, ga.l.small), 256, 0, s>>>(ga);
    const Prod kind = pick_prod(q.d);
    if (kind == Prod::kBig)
      run_prod<DT, ODT, Big, SPLIT>(q, p, wv, dz, v0, nv, 1.f / raise, dw, s);
    else if (kind == Prod::kHalf)
      run_prod<DT, ODT, Half, SPLIT>(q, p, wv, dz, v0, nv, 1.f / raise, dw, s);
    else
      run_prod<DT, ODT, Quarter, SPLIT>(q, p, wv, dz, v0, nv, 1.f / raise, dw, s);
    if (int rc = check_launch("pdh_linear_xent_bwd"); rc != PDH_OK) return rc;
  }
  xent_sum<ODT><<<dim3(blocks_for(q.n * (dp / 4))), 256, 0, s>>>(p.parts, dx, q.n, static_cast<int>(q.d), dp, q.n * dp,
                                                                static_cast<int>(p.slices.x), p.most, 1.f / raise, targets, q.v,
                                                                ignore);
  return check_launch("pdh_linear_xent_bwd (dx)");
}

}  // namespace
}  // namespace pdh

using namespace pdh;

extern "C" size_t pdh_linear_xent_workspace(const void* x, const void* w, int64_t tokens, int64_t width, int64_t vocab,
                                            int64_t ldx, int64_t ldw, int dtype, int backward) {
  if (check("pdh_linear_xent_workspace", tokens, width, vocab, ldx, ldw, dtype) != PDH_OK || tokens == 0) return 0;
  const Problem q{tokens, width, vocab, ldx, ldw, x, w, dtype};
  const bool fx = Problem::fit(x, ldx, width, dtype), fw = Problem::fit(w, ldw, width, dtype);
  Space ws{nullptr};
  if (backward)
    plan_bwd(q, ws, fw);
  else
    plan_fwd(q, ws, fx, fw);
  return ws.used;
}

extern "C" int pdh_linear_xent_fwd(const void* x, const void* w, const int64_t* targets, float* loss, float* lse,
                                   int64_t tokens, int64_t width, int64_t vocab, int64_t ldx, int64_t ldw,
                                   int64_t ignore_index, int dtype, int* bad, void* ws, size_t ws_bytes, void* stream) {
  if (int rc = check("pdh_linear_xent_fwd", tokens, width, vocab, ldx, ldw, dtype); rc != PDH_OK) return rc;
  if (tokens == 0) return PDH_OK;
  PDH_REQUIRE(x && w && targets && loss && lse, PDH_EINVAL, "pdh_linear_xent_fwd: null pointer");
  const Problem q{tokens, width, vocab, ldx, ldw, x, w, dtype};
  const bool fx = Problem::fit(x, ldx, width, dtype), fw = Problem::fit(w, ldw, width, dtype);
  Space space{static_cast<char*>(ws)};
  const FwdPlan p = plan_fwd(q, space, fx, fw);
  PDH_REQUIRE(ws && aligned16(ws) && ws_bytes >= space.used, PDH_EINVAL,
              "pdh_linear_xent_fwd: the workspace holds %zu bytes, %zu are needed, 16-byte aligned", ws ? ws_bytes : size_t{0},
              space.used);
  hipStream_t s = as_stream(stream);
  if (dtype == PDH_F32) return run_fwd<PDH_BF16, true>(q, p, targets, ignore_index, loss, lse, bad, s);
  if (dtype == PDH_BF16) return run_fwd<PDH_BF16, false>(q, p, targets, ignore_index, loss, lse, bad, s);
  return run_fwd<PDH_F16, false>(q, p, targets, ignore_index, loss, lse, bad, s);
}

extern "C" int pdh_linear_xent_bwd(const void* x, const void* w, const int64_t* targets, const float* lse,
                                   const float* dloss, void* dx, void* dw, int64_t tokens, int64_t width, int64_t vocab,
                                   int64_t ldx, int64_t ldw, int64_t ignore_index, int dtype, void* ws, size_t ws_bytes,
                                   void* stream) {
  if (int rc = check("pdh_linear_xent_bwd", tokens, width, vocab, ldx, ldw, dtype); rc != PDH_OK) return rc;
  PDH_REQUIRE(tokens > 0, PDH_EINVAL, "pdh_linear_xent_bwd: no tokens");
  PDH_REQUIRE(x && w && targets && lse && dloss && dx && dw, PDH_EINVAL, "pdh_linear_xent_bwd: null pointer");
  const Problem q{tokens, width, vocab, ldx, ldw, x, w, dtype};
  const bool fw = Problem::fit(w, ldw, width, dtype);
  Space space{static_cast<char*>(ws)};
  const BwdPlan p = plan_bwd(q, space, fw);
  PDH_REQUIRE(ws && aligned16(ws) && ws_bytes >= space.used, PDH_EINVAL,
              "pdh_linear_xent_bwd: the workspace holds %zu bytes, %zu are needed, 16-byte aligned", ws ? ws_bytes : size_t{0},
              space.used);
  hipStream_t s = as_stream(stream);
  if (dtype == PDH_F32) return run_bwd<PDH_BF16, PDH_F32, true>(q, p, targets, lse, dloss, ignore_index, dx, dw, s);
  if (dtype == PDH_BF16) return run_bwd<PDH_BF16, PDH_BF16, false>(q, p, targets, lse, dloss, ignore_index, dx, dw, s);
  return run_bwd<PDH_F16, PDH_F16, false>(q, p, targets, lse, dloss, ignore_index, dx, dw, s);
}
