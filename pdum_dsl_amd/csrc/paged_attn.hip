// Attention over a paged cache: rows of several sequences, causal, with an optional window and first tokens kept.
//
//   x(p, s) = scale q_p . k_s over the visible s: s <= p and (s < sinks or s > p - window)
//   o = sum_s softmax(x) v_s, lse = log sum_s exp x;  a row with no visible key: o = 0, lse = -inf
//
// Two kernels, by the mean number of rows of a sequence times the group of query heads on a key/value head: to 16 of them
// the decode kernel (bytes bound it), above the prompt kernel (matrix products do). 64 sequences of 8192 tokens, 32/8 heads
// of 128, us by the one / the other: 4 rows each 367 / 403 (4 bits 128 / 222), 5 rows, two blocks, 711 / 421 (239 / 233). The
// switch lies where 16 bits have it; 4 bits, whose bytes take 107 us, jump there (8 rows 226, 16 275). Both take any batch, the
// whole of it by its mean. Single tokens that a prompt brings to the prompt kernel cost what they read in 16 bits (64 of 8192
// tokens and a prompt of 2048: 421 together, 361 + 64 apart), more in 4 (282, 105 + 69); a piece that single tokens bring to
// the decode kernel reads its cache once for 16 of its rows times the group: 255 of 1000 tokens and 500 rows over 32768, 2403
// together, 189 + 282 apart (4 bits 807, 59 + 286).
#include "attn_common.h"
#include "paged.h"

#include <atomic>
#include <cmath>

namespace pdh {
namespace {

constexpr float kInf = __builtin_inff();

// Softmax weights are factors of a 16-bit matrix product, which has no wider ones, rounded to the type (half a step of each;
// their sum is of the fp32 ones). A second product by what the rounding leaves would bring o to 64 bits' own rounding: half
// as many matrix instructions again in prompts, which they bound; in decode 4% for four drafted tokens of 4 bits and 7% for
// heads of 64, and a visible infinity times a rest of 0 or less is not its sum. f16 ends at 2^-24: there weights are taken
// 2^kLift larger, o and the sum with them, so that the largest is 2^7 to 2^15 and what is lost lies under 2^-32 of it: 2^20
// keys of that come to 2^-12. States are (m, l, o) with m - kLift for m.
template <typename T>
constexpr float kLift = std::is_same_v<T, _Float16> ? 7.0f : 0.0f;

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
  // The page of an entry is read without a branch, entries past the table's as its last (their keys are past reach and
  // seen by no row), and looked at only when it is needed, so that the load is not waited for before.
  const int32_t* table;  // some memory where the table has no entry
  int last_entry, pages;
  __device__ __forceinline__ bool has(int page) const {
    return static_cast<uint32_t>(page) < static_cast<uint32_t>(pages);
  }
};

// One row by one wave: keys 64 at a time, one a lane; the online softmax's maximum and sum are the wave's, o's features lie
// across its lanes. It touches no key that the row does not see, which makes it the way out for rows that share blocks of keys
// with values that are not finite and not theirs. The row's softmax state over the visible keys of [k0, k1): m in units of
// log2, o unnormalised, features lane + 64 j.
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
    const int64_t kat = seen ? pool_at<BITS>(a.c, page, key & mask) + hk * a.c.sh : 0;
    const int64_t ksat = seen ? scale_at(a.c, page, key & mask) + hk * a.c.ssh : 0;
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
      const int64_t at = (static_cast<int64_t>(__shfl(static_cast<int>(kat >> 32), kk, kWave)) << 32) |
                         static_cast<uint32_t>(__shfl(static_cast<int>(kat), kk, kWave));
      if constexpr (BITS == 16) {
        const uint16_t* v = static_cast<const uint16_t*>(a.c.v) + at;
#pragma unroll
        for (int j = 0; j < D / 64; ++j) o[j] = __builtin_fmaf(pk, Elem<T>::to_f32(v[lane + 64 * j]), o[j]);
      } else {
        const int64_t sat = (static_cast<int64_t>(__shfl(static_cast<int>(ksat >> 32), kk, kWave)) << 32) |
                            static_cast<uint32_t>(__shfl(static_cast<int>(ksat), kk, kWave));
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

// A finished row: o's features lane + 64 j, m in units of log2.
template <typename T, int D>
__device__ __forceinline__ void write_row(const PagedAttn& a, int row, int h, float m, float l, const float (&o)[D / 64]) {
  const int lane = threadIdx.x & 63;
  const float inv = l == 0.f ? 0.f : 1.0f / l;  // nothing seen, or scores of -inf alone
  uint16_t* out = a.o + row * a.o_st + h * a.o_sh;
#pragma unroll
  for (int j = 0; j < D / 64; ++j) out[lane + 64 * j] = Elem<T>::from_f32(o[j] * inv);
  if (lane == 0 && a.lse) a.lse[static_cast<int64_t>(row) * a.heads_q + h] = l == 0.f ? -kInf : (m + __log2f(l)) * kLn2;
}

// ------------------------------------------------------------------ few rows a sequence
//
// Decode: the work is reading the caches once. A sequence's rows times the group of query heads that share a key/value head,
// flattened (row * group + head), are cut into blocks of 16, the columns of v_mfma_f32_16x16x32: every cached byte that a
// block reads serves all of them. Keys go by blocks of 32 on the absolute grid, so that a block lies in at most two pages,
// whose numbers are wave-uniform scalars, fetched a block before its loads are issued.
//
// Memory bounds it. 64 x 8192 tokens, 32/8 heads of 128: 16 bits 360 us, 2154 MB fetched (6.0 TB/s), 4 bits 107 us, 607 MB
// (5.7; 36 MB of them lines of scales that a page of 16 rows fills by half); with every sequence on the same pages, which L2
// then holds, 4 bits take 71. A copy of such sizes moves 5.1 to 5.4 TB/s. 24 ragged sequences of up to 30000 under a window:
// 75 us, 411 MB. Short calls are latency: 1 x 1000 tokens 9.4 us, of which two rounds of blocks are half.
//
// Shares. Sequences differ in length, and the lengths are device memory. Every workgroup sums up all sequences' work (blocks of
// keys x blocks of rows x heads), takes the same share of the line they form, and sweeps what lies in it: a part of one
// (sequence, head, row block), several whole ones, a part of another. A whole one is written out at once; of a cut one each
// workgroup leaves its state (m, l, o) and paged_decode_merge, one workgroup for each, joins them.
//
// A block of keys (S^T = K Q^T, O^T += V^T P^T as in decode.hip): K straight from its loads as the A operand, V through a
// tile of the wave's own in LDS, read back transposed. The next block's loads are in flight while one is computed. A 4-bit row
// is loaded as codes: a lane takes features D/4 g .. + D/4 of its row (one load, one scale), which k-step s contracts by
// eights, and q is laid out to match; V is widened to 16 bits on its way into LDS.

// Workgroups a compute unit holds at once: what keeps memory busy, no more. 64 sequences of 8192 tokens, 32/8 heads, us with
// two / three: 4 bits, D = 128, 126 / 130, D = 64 59 / 64; 16 bits, 16 heads of 64, 378 / 376; D = 128 has registers for two.
template <int D, int BITS>
__host__ __device__ constexpr int dec_wgs() {
  return BITS == 16 && D == 64 ? 3 : 2;
}

template <int D, int BITS>
struct DecCfg {
  static constexpr int KS = D / 32;        // k-steps of the score product
  static constexpr int ET = D / 16;        // 16-feature tiles of the output product
  static constexpr int CPR = D / 8;        // 16-byte chunks a 16-bit row
  static constexpr int RPI = 64 / CPR;     // rows a 16-bit value load
  static constexpr int VL = 32 / RPI;      // 16-bit value loads a block
  static constexpr int VROW = D * 2 + 32;  // LDS bytes a value row (32 of padding: conflict-free transposed reads)
  static constexpr int VTILE = 32 * VROW;
  static constexpr int RS = 2 + D;  // floats of a row's state: m, l, o
  static constexpr int RED = 4 * 16 * RS * 4;
  static constexpr int LDS = 4 * VTILE > RED ? 4 * VTILE : RED;
  // Blocks of keys in registers: one computed, the others in flight. Three and four, 4 bits, 64 x 8192, heads of 128: 128 and
  // 130 us against 126; one, refilled when its keys are used, 125, but heads of 64 64 against 59.
  static constexpr int NB = 2;
  // The unit of work is a block of keys. An item costs ITEM more (what its q, its state and their join take), so that the
  // short ones of a batch of many are not all one workgroup's; a share is at least LEAST, two rounds of the four waves, and
  // ITEM as much, so that no short share sweeps keys of two items, one after the other. us at ITEM 0 / 4 / 8 / 12: 7 x 4 tokens over
  // 5003 (4 bits, heads of 64) 17.7 / 17.5 / 16.4 / 16.1, 1 over 5000 16.2 / 14.1 / 12.9 / 12.9, 4 over 300 15.2 / 13.1 / 11.8 /
  // 11.9, 512 ragged over 100 64.5 / 56.0 / 57.5 / 58.5, 24 over 30000 under a window 82 / 80 / 80 / 83; at LEAST 4 / 8 / 16,
  // 1 over 1000 11.2 / 11.7 / 15.7, 1 over 5000 15.3 / 12.9 / 16.2.
  static constexpr int ITEM = 8, LEAST = 8;
};

// One block of 32 keys in flight.
template <int D, int BITS>
struct DecBlk;
template <int D>
struct DecBlk<D, 16> {
  u32x4 k[2 * D / 32], v[32 / (64 / (D / 8))];
};
template <int D>
struct DecBlk<D, 4> {
  typedef uint32_t codes __attribute__((ext_vector_type(D / 32)));
  codes k[2], v[2];
  uint32_t ks[2], vs[2];  // scale bytes
};

// A resource over wave-uniform memory whose address the compiler may hold in vector registers.
__device__ __forceinline__ rsrc_t uniform_rsrc(const void* base, uint32_t bytes) {
  const uint64_t u = reinterpret_cast<uintptr_t>(base);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(u));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(u >> 32));
  return make_rsrc(reinterpret_cast<const void*>(static_cast<uint64_t>(hi) << 32 | lo), __builtin_amdgcn_readfirstlane(bytes));
}

__device__ __forceinline__ uint32_t bload8(rsrc_t r, uint32_t voff, uint32_t soff) {
  return __builtin_amdgcn_raw_buffer_load_b8(r, voff, soff, 0);
}
template <int D>
__device__ __forceinline__ typename DecBlk<D, 4>::codes bload_codes(rsrc_t r, uint32_t voff, uint32_t soff) {
  if constexpr (D == 128)
    return bload128(r, voff, soff);
  else
    return bload64(r, voff, soff);
}

// Device memory that no kernel in flight writes, read through the scalar cache where the address is uniform.
__device__ __forceinline__ int32_t uniform_i32(const int32_t* p) {
  typedef const __attribute__((address_space(4))) int32_t c_i32;
  return *(c_i32*)(p);
}

// A sequence's work: blocks of rows and of keys. Visible keys lie in blocks [0, sb) (the first tokens) and [wb, eb).
struct SeqPlan {
  int row0, n, pos0;  // first row, rows, the first row's position
  int nb, sb, wb, blocks;
  __device__ __forceinline__ int key_block(int v) const { return v < sb ? v : v - sb + wb; }
};

__device__ __forceinline__ int scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }

__device__ __forceinline__ int64_t scalar64(int64_t x) {
  return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(scalar(static_cast<int>(x >> 32)))) << 32 |
                              static_cast<uint32_t>(scalar(static_cast<int>(x))));
}

template <int ROWS>
__device__ __forceinline__ SeqPlan plan_of(const PagedAttn& a, int i) {
  Seq s{0, 0, 0};
  if (i < a.b.seqs) {
    s = seq_at(a.b, i);
  } else if (a.zero_rest) {  // the rows behind the last sequence: no keys
    const int r0 = a.b.seqs ? clamp_row(a.b.starts[i], static_cast<int>(a.b.rows)) : 0;
    s = Seq{r0, static_cast<int>(a.b.rows) - r0, 0};
  }
  SeqPlan p;
  p.row0 = s.row0;
  p.n = s.n;
  p.pos0 = s.len - s.n;
  const int end = s.len < a.reach ? s.len : a.reach;
  const int eb = (end + 31) / 32;
  const int lo = p.pos0 - a.window + 1;
  p.wb = lo > 0 ? lo / 32 : 0;
  p.wb = p.wb < eb ? p.wb : eb;
  const int sink = a.sinks < end ? a.sinks : end;
  p.sb = (sink + 31) / 32;
  p.sb = p.sb < p.wb ? p.sb : p.wb;
  p.blocks = p.sb + eb - p.wb;
  p.blocks = p.blocks > 0 ? p.blocks : 1;  // one that sees nothing
  p.nb = static_cast<int>((static_cast<int64_t>(s.n) * a.group + ROWS - 1) / ROWS);
  return p;
}

// The plan of a wave-uniform sequence, held in scalar registers.
template <int ROWS>
__device__ __forceinline__ SeqPlan uniform_plan(const PagedAttn& a, int i) {
  const SeqPlan p = plan_of<ROWS>(a, i);
  return SeqPlan{scalar(p.row0), scalar(p.n), scalar(p.pos0), scalar(p.nb), scalar(p.sb), scalar(p.wb), scalar(p.blocks)};
}

// An item that starts in a workgroup's share and ends in another's (last; -1: none): its first row, rows, number of
// flattened rows before it, head.
struct DecMeta {
  int last, row0, rows, f0, head;
};

// FAR: a pool reaches past the offsets of one buffer resource (2^31 bytes), and each page gets its own: 64 x 8192 tokens of 16
// bits take as long so (376 us), but 2 x 4096 tokens of a prompt 264 instead of 260.
template <typename T, int D, int BITS, bool FAR>
__global__ __launch_bounds__(256, (dec_wgs<D, BITS>())) void paged_decode(PagedAttn a, DecMeta* meta, float* ws) {
  using C = DecCfg<D, BITS>;
  constexpr int KS = C::KS, ET = C::ET, RS = C::RS;
  __shared__ __attribute__((aligned(1024))) unsigned char dsm[C::LDS];
  __shared__ int64_t scan[4];
  struct Start {
    SeqPlan sp;
    int seq, item, unit;
  };
  __shared__ Start first;
  const int tid = threadIdx.x, lane = tid & 63, w = wave_id();
  const int col = lane & 15, g = lane >> 4;
  const int hkv = static_cast<int>(a.c.heads), R = a.group;

  // ---- this workgroup's share [at, at + left) of the line of (sequence, head, row block, units of it)
  const int nseq = static_cast<int>(a.b.seqs);
  const int each = (nseq + 255) / 256;
  auto cost = [&](const SeqPlan& p) { return static_cast<int64_t>(p.nb) * (p.blocks + C::ITEM) * hkv; };
  SeqPlan mp{};
  int64_t mine = 0;
  for (int j = 0; j < each; ++j) {
    const int i = tid * each + j;
    if (i < nseq) {
      mp = plan_of<16>(a, i);
      mine += cost(mp);
    }
  }
  int64_t incl = mine;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t o = (static_cast<int64_t>(__shfl_up(static_cast<int>(incl >> 32), off, kWave)) << 32) |
                      static_cast<uint32_t>(__shfl_up(static_cast<int>(incl), off, kWave));
    incl += lane >= off ? o : 0;
  }
  if (lane == 63) scan[w] = incl;
  __syncthreads();
  int64_t total = 0, before = incl - mine;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    before += i < w ? scan[i] : 0;
    total += scan[i];
  }
  total = scalar64(total);
  int64_t per = scalar64((total + gridDim.x - 1) / gridDim.x);
  per = per > C::LEAST ? (per + 3) / 4 * 4 : C::LEAST;  // whole rounds of the four waves
  int64_t at = per * blockIdx.x;
  int64_t left = total - at < per ? total - at : per;
  if (left <= 0) {
    if (tid == 0) meta[blockIdx.x] = DecMeta{-1, 0, 0, 0, 0};
    return;
  }
  if (before <= at && at < before + mine) {  // the share starts in one of this thread's sequences
    int64_t in = at - before;
    int i = tid * each;
    if (each > 1)
      for (mp = plan_of<16>(a, i); in >= cost(mp); mp = plan_of<16>(a, ++i)) in -= cost(mp);
    const int units = mp.blocks + C::ITEM;
    first = Start{mp, i, static_cast<int>(in / units), static_cast<int>(in % units)};
  }
  __syncthreads();
  SeqPlan sp{scalar(first.sp.row0), scalar(first.sp.n),  scalar(first.sp.pos0),  scalar(first.sp.nb),
             scalar(first.sp.sb),   scalar(first.sp.wb), scalar(first.sp.blocks)};
  int seq = scalar(first.seq), item = scalar(first.item), unit = scalar(first.unit);  // heads x row blocks < 2^31 (host)
  DecMeta cut{-1, 0, 0, 0, 0};

  unsigned char* vt = dsm + w * C::VTILE;
  // transposed value reads: lane 4k + c of group g addresses row 4 g + k, features 4 c .. +3 (+ 16 t)
  const int trb = (4 * g + (col >> 2)) * C::VROW + (col & 3) * 8;
  constexpr int ES = BITS == 16 ? 2 : 1;  // bytes of a stride's unit
  const uint32_t rst = static_cast<uint32_t>(a.c.sr) * ES, srst = static_cast<uint32_t>(a.c.ssr);
  const int vrow = BITS == 16 ? lane / C::CPR : lane / 4, vch = BITS == 16 ? lane % C::CPR : lane % 4;

  while (left > 0) {
    const int rb = scalar(item % sp.nb), head = scalar(item / sp.nb);
    const int units = sp.blocks + C::ITEM - unit;  // to the item's end
    const int take = scalar(static_cast<int>(units < left ? units : left));
    const int kb = unit > C::ITEM ? unit - C::ITEM : 0, k_end = unit + take > C::ITEM ? unit + take - C::ITEM : 0;
    if (k_end == 0) break;  // the share ends before the item's first key

    // ---- the block's rows: column c is flattened row 16 rb + c
    const int f0 = rb * 16, nq = sp.n * R - f0 < 16 ? sp.n * R - f0 : 16;  // rows x heads_q < 2^31
    const int fc = f0 + (col < nq ? col : 0);
    const int pos = sp.pos0 + fc / R;
    const int pos_lo = scalar(sp.pos0 + f0 / R), pos_hi = scalar(sp.pos0 + (f0 + nq - 1) / R);
    u32x4 qb[KS];
    {
      const uint16_t* qr = a.q + (sp.row0 + fc / R) * a.q_st + (head * R + fc % R) * a.q_sh;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(qr + (BITS == 16 ? s * 32 + g * 8 : g * (D / 4) + s * 8));
        qb[s] = col < nq ? v : u32x4{0u, 0u, 0u, 0u};
      }
    }

    struct Pages {
      int p[2];  // the entries of a block's two halves, as they stand in the table
    };
    const int32_t* trow = a.table + seq * a.b.ld_table;
    auto pages = [&](int v) {
      const int key0 = scalar(sp.key_block(v) * 32);
      const int e0 = key0 >> a.shift, e1 = (key0 + 16) >> a.shift;
      return Pages{{uniform_i32(trow + (e0 < a.last_entry ? e0 : a.last_entry)),
                    uniform_i32(trow + (e1 < a.last_entry ? e1 : a.last_entry))}};
    };
    const char* const kpool = static_cast<const char*>(a.c.k) + head * a.c.sh * ES;
    const char* const vpool = static_cast<const char*>(a.c.v) + head * a.c.sh * ES;
    const char* const kspool = static_cast<const char*>(a.c.k_scale) + head * a.c.ssh;
    const char* const vspool = static_cast<const char*>(a.c.v_scale) + head * a.c.ssh;
    // Through buffer resources, a lane's address one 32-bit offset: one resource a pool and a page's place as the scalar
    // offset, or FAR, a resource a page. A half without a page reads page 0: what it holds is masked.
    const int in_last = (1 << a.shift) - 1;
    const uint32_t whole_span = (a.pages - 1) * (static_cast<uint32_t>(a.c.sp) * ES) + in_last * rst + D * BITS / 8;
    const uint32_t whole_sspan = (a.pages - 1) * static_cast<uint32_t>(a.c.ssp) + in_last * srst + D / 32;
    rsrc_t krs = make_rsrc(kpool, whole_span), vrs = make_rsrc(vpool, whole_span);
    rsrc_t ksrs = make_rsrc(kspool, whole_sspan), vsrs = make_rsrc(vspool, whole_sspan);
    auto load = [&](int v, const Pages& pg, DecBlk<D, BITS>& r) {
      const int key0 = scalar(sp.key_block(v) * 32);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int p = a.has(pg.p[h]) ? pg.p[h] : 0;
        const int in = (key0 + 16 * h) & in_last;
        uint32_t so = 0, sso = 0;
        if constexpr (FAR) {
          const int64_t at = pool_at<BITS>(a.c, p, in) * ES;
          const uint32_t span = 15 * rst + D * BITS / 8;
          krs = uniform_rsrc(kpool + at, span);
          vrs = uniform_rsrc(vpool + at, span);
          if constexpr (BITS == 4) {
            const int64_t sat = scale_at(a.c, p, in);
            const uint32_t sspan = 15 * srst + D / 32;
            ksrs = uniform_rsrc(kspool + sat, sspan);
            vsrs = uniform_rsrc(vspool + sat, sspan);
          }
        } else {
          so = p * (static_cast<uint32_t>(a.c.sp) * ES) + in * rst;
          if constexpr (BITS == 4) sso = p * static_cast<uint32_t>(a.c.ssp) + in * srst;
        }
        if constexpr (BITS == 16) {
#pragma unroll
          for (int s = 0; s < KS; ++s) r.k[h * KS + s] = bload128(krs, col * rst + g * 16 + s * 64, so);
#pragma unroll
          for (int j = 0; j < C::VL / 2; ++j)
            r.v[h * (C::VL / 2) + j] = bload128(vrs, vrow * rst + vch * 16, so + j * C::RPI * rst);
        } else {
          r.k[h] = bload_codes<D>(krs, col * rst + g * (D / 8), so);
          r.ks[h] = bload8(ksrs, col * srst + g * (D / 4) / 32, sso);
          r.v[h] = bload_codes<D>(vrs, vrow * rst + vch * (D / 8), so);
          r.vs[h] = bload8(vsrs, vrow * srst + vch * (D / 4) / 32, sso);
        }
      }
    };

    // blocks [c0, c1) are seen whole by every row, as far as their pages are there
    int c0, c1;
    {
      const int edge = pos_hi - a.window + 1;
      const int first = edge > 0 ? (edge + 31) / 32 : 0, last = (pos_lo + 1 < a.reach ? pos_lo + 1 : a.reach) >> 5;
      c0 = sp.sb + (first > sp.wb ? first - sp.wb : 0);
      c1 = sp.sb + (last > sp.wb ? last - sp.wb : 0);
    }

    float m = -kInf, lsum = 0.f;  // the raw scores' reference, this lane's part of the sum
    f32x4 o[ET];
#pragma unroll
    for (int t = 0; t < ET; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};

    auto block = [&](int v, const Pages& pg, DecBlk<D, BITS>& r) __attribute__((always_inline)) {
      const int key0 = scalar(sp.key_block(v) * 32);
      const bool full = (v >= c0) & (v < c1) & a.has(pg.p[0]) & a.has(pg.p[1]);  // every row sees every key
      if (!full) {  // keys that no row sees: their values count as zero
        const int last = (pos_hi < a.reach ? pos_hi : a.reach - 1) - key0, first = pos_lo - a.window + 1 - key0;
        const int kept = a.sinks - key0;
        auto gone = [&](int at, int p) { return !a.has(p) | (at > last) | ((at >= kept) & (at < first)); };
        if constexpr (BITS == 16) {
#pragma unroll
          for (int j = 0; j < C::VL; ++j)
            if (gone(j * C::RPI + vrow, pg.p[j / (C::VL / 2)])) r.v[j] = u32x4{0u, 0u, 0u, 0u};
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (gone(16 * h + vrow, pg.p[h])) {
              r.v[h] = typename DecBlk<D, 4>::codes{};
              r.vs[h] = 0;
            }
        }
      }
      // values -> this wave's tile, rows of keys
      if constexpr (BITS == 16) {
#pragma unroll
        for (int j = 0; j < C::VL; ++j) *reinterpret_cast<u32x4*>(vt + (j * C::RPI + vrow) * C::VROW + vch * 16) = r.v[j];
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < KS; ++i)
            *reinterpret_cast<u32x4*>(vt + (16 * h + vrow) * C::VROW + vch * (D / 2) + i * 16) =
                fp4_row8<T>(r.v[h][i], e8m0(r.vs[h]));
      }
      // S^T: keys key0 + 16 h + 4 g + i (accumulator i), row col
      f32x4 sc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          u32x4 kk;
          if constexpr (BITS == 16)
            kk = r.k[h * KS + s];
          else
            kk = fp4_row8<T>(r.k[h][s], e8m0(r.ks[h]));
          sc[h] = mfma16<T>(kk, qb[s], sc[h]);
        }
      if (!full) {
        const int kl = key0 + 4 * g;
        const int last = (pos < a.reach ? pos : a.reach - 1) - kl, first = pos - a.window + 1 - kl, kept = a.sinks - kl;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int cc = 16 * (i >> 2) + (i & 3);
          const int end = a.has(pg.p[i >> 2]) ? last : -1 - kMaxTokens;
          const bool seen = (cc <= end) & ((cc >= first) | (cc < kept));
          sc[i >> 2][i & 3] = seen ? sc[i >> 2][i & 3] : -kInf;
        }
      }
      // The exponentials refer to a maximum that moves only when they leave (0, 2^(8 + kLift)], or are not numbers (a maximum of
      // -inf: the first block): then the block's maximum is found and everything rescaled.
      u32x4 pb;
      auto expo = [&](float ref) {
        const float mc = ref * a.c2 - kLift<T>;
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = fast_exp2(__builtin_fmaf(sc[i >> 2][i & 3], a.c2, -mc));
        pb = u32x4{pack2<T>(p[0], p[1]), pack2<T>(p[2], p[3]), pack2<T>(p[4], p[5]), pack2<T>(p[6], p[7])};
        return ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
      };
      constexpr float kLimit = kLift<T> > 0.f ? 32768.f : 256.f;
      float part = expo(m);
      if (__builtin_amdgcn_ballot_w64(!(part <= kLimit)) != 0) {
        float mx = sc[0][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) mx = fmaxf(mx, sc[i >> 2][i & 3]);
        const float mnew = fmaxf(m, max4g(mx));
        const float ref = mnew == -kInf ? 0.f : mnew;  // scores of -inf alone weigh 0, not NaN
        const float alpha = mnew == m ? 1.f : fast_exp2((m - ref) * a.c2);
        lsum *= alpha;
#pragma unroll
        for (int t = 0; t < ET; ++t) o[t] *= alpha;
        m = mnew;
        part = expo(ref);
      }
      lsum += part;
#pragma unroll
      for (int t = 0; t < ET; ++t) {
        const u32x2 lo = ds_read_tr16(vt + trb + 32 * t);
        const u32x2 hi = ds_read_tr16(vt + trb + 16 * C::VROW + 32 * t);
        o[t] = mfma16<T>(u32x4{lo.x, lo.y, hi.x, hi.y}, pb, o[t]);
      }
    };

    // Each wave takes every fourth block. Past its last one the loads in flight re-read that block (an L2 hit): they are
    // issued whatever comes, so that the compiler's wait counts stay exact.
    if (kb + w < k_end) {
      const int v_last = kb + w + (k_end - 1 - kb - w) / 4 * 4;
      auto bound = [&](int v) { return v < v_last ? v : v_last; };
      constexpr int NB = C::NB;
      DecBlk<D, BITS> r[NB];
      Pages pg[NB], next = pages(kb + w);
      int v = kb + w, ahead = v;
      auto fetch = [&](int i) __attribute__((always_inline)) {
        load(ahead, next, r[i]);
        pg[i] = next;
        ahead = bound(ahead + 4);
        next = pages(ahead);
      };
#pragma unroll
      for (int i = 0; i < NB - 1; ++i) fetch(i);
      // (not left in the middle of a round: the accumulators would be held twice)
#pragma unroll 1
      for (; v < k_end; v += 4 * NB) {
#pragma unroll
        for (int i = 0; i < NB; ++i)
          if (i == 0 || v + 4 * i < k_end) {
            fetch((i + NB - 1) % NB);
            block(v + 4 * i, pg[i], r[i]);
          }
      }
    }
    lsum = sum4g(lsum);

    // ---- the four waves' states meet in LDS, over the value tiles
    __syncthreads();
    float* red = reinterpret_cast<float*>(dsm);
    if (col < nq) {
      float* rec = red + (w * 16 + col) * RS;
      if (g == 0) {
        rec[0] = m * a.c2 - kLift<T>;  // log2 units
        rec[1] = lsum;
      }
#pragma unroll
      for (int t = 0; t < ET; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) rec[2 + 16 * t + 4 * g + i] = o[t][i];
    }
    __syncthreads();
    const bool whole = k_end - kb == sp.blocks;
    float* rec = ws + (static_cast<int64_t>(blockIdx.x) * 2 + (kb == 0 ? 1 : 0)) * 16 * RS;
    for (int c = w; c < nq; c += 4) {
      float mw[4], mm = -kInf, l = 0.f, acc[D / 64] = {};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mw[i] = red[(i * 16 + c) * RS];
        mm = fmaxf(mm, mw[i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float* p = red + (i * 16 + c) * RS;
        const float f = mw[i] == -kInf ? 0.f : fast_exp2(mw[i] - mm);
        l += f * p[1];
#pragma unroll
        for (int j = 0; j < D / 64; ++j) acc[j] += f * p[2 + lane + 64 * j];
      }
      const int f = f0 + c, tok = f / R, hq = head * R + f % R;
      if (pos_lo != pos_hi) {
        // Rows at different positions share blocks of keys: 0 times a value that only some of them see is NaN where it is
        // an infinity or a NaN. Such a row is done again, by itself.
        bool nan = l != l;
#pragma unroll
        for (int j = 0; j < D / 64; ++j) nan |= acc[j] != acc[j];
        if (__builtin_amdgcn_ballot_w64(nan) != 0) {
          mm = -kInf;
          l = 0.f;
#pragma unroll
          for (int j = 0; j < D / 64; ++j) acc[j] = 0.f;
          const uint16_t* qr = a.q + (sp.row0 + tok) * a.q_st + hq * a.q_sh;
          const int s1 = (k_end < sp.sb ? k_end : sp.sb) * 32;
          if (kb < sp.sb) row_sweep<T, D, BITS>(a, seq, head, qr, sp.pos0 + tok, kb * 32, s1, mm, l, acc);
          if (k_end > sp.sb)
            row_sweep<T, D, BITS>(a, seq, head, qr, sp.pos0 + tok, sp.key_block(kb > sp.sb ? kb : sp.sb) * 32,
                                  sp.key_block(k_end - 1) * 32 + 32, mm, l, acc);
        }
      }
      if (whole) {
        write_row<T, D>(a, sp.row0 + tok, hq, mm, l, acc);
      } else {
        if (lane == 0) {
          rec[c * RS] = mm;
          rec[c * RS + 1] = l;
        }
#pragma unroll
        for (int j = 0; j < D / 64; ++j) rec[c * RS + 2 + lane + 64 * j] = acc[j];
      }
    }
    if (kb == 0 && !whole)
      cut = DecMeta{static_cast<int>((at + units - 1) / per), sp.row0, nq, f0, head};
    __syncthreads();  // before the next item's tiles

    left -= take;
    at += take;
    unit += take;
    if (take == units && left > 0) {
      unit = 0;
      ++item;
      if (item == sp.nb * hkv) {
        item = 0;
        do sp = uniform_plan<16>(a, ++seq);
        while (sp.n == 0);
      }
    }
  }
  if (tid == 0) meta[blockIdx.x] = cut;
}

// Joins a cut item's states: the workgroup that the item starts in left the first in its second record, the others up to
// `last` theirs in their first. Eight waves: four rows at a time, half of the records each, eight of them in flight; the
// halves meet in LDS. Then the rows of no sequence, before the first and behind the last, spread over the grid. 5 us at 64 x
// 8192 tokens (as many workgroups as the decode kernel's, which 1024 threads each would run in two rounds: 8).
template <typename T, int D>
__global__ __launch_bounds__(512) void paged_decode_merge(PagedAttn a, const DecMeta* meta, const float* ws) {
  constexpr int RS = 2 + D, DL = D / 64;
  __shared__ float part[8][RS];
  const DecMeta c = meta[blockIdx.x];
  const int lane = threadIdx.x & 63, w = wave_id();
  if (c.last >= 0) {
    const int nrec = c.last - static_cast<int>(blockIdx.x) + 1;
    for (int i0 = 0; i0 < c.rows; i0 += 4) {
      const int i = i0 + (w >> 1);
      float m = -kInf, l = 0.f, o[DL] = {};
      if (i < c.rows) {
        for (int r0 = w & 1; r0 < nrec; r0 += 16) {
          float rm[8], rl[8], ro[8][DL];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const bool in = r0 + 2 * j < nrec;  // one that is not there reads another's place, and counts as empty
            const int r = in ? r0 + 2 * j : r0;
            const float* p = ws + ((static_cast<int64_t>(blockIdx.x) + r) * 2 + (r == 0)) * 16 * RS + i * RS;
            rm[j] = in ? p[0] : -kInf;
            rl[j] = in ? p[1] : 0.f;
#pragma unroll
            for (int d = 0; d < DL; ++d) {
              const float x = p[2 + lane + 64 * d];
              ro[j][d] = in ? x : 0.f;
            }
          }
          float mm = m;
#pragma unroll
          for (int j = 0; j < 8; ++j) mm = fmaxf(mm, rm[j]);
          const float f0 = m == -kInf ? 0.f : fast_exp2(m - mm);
          l *= f0;
#pragma unroll
          for (int d = 0; d < DL; ++d) o[d] *= f0;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float f = rm[j] == -kInf ? 0.f : fast_exp2(rm[j] - mm);
            l += f * rl[j];
#pragma unroll
            for (int d = 0; d < DL; ++d) o[d] += f * ro[j][d];
          }
          m = mm;
        }
      }
      if (lane == 0) {
        part[w][0] = m;
        part[w][1] = l;
      }
#pragma unroll
      for (int d = 0; d < DL; ++d) part[w][2 + lane + 64 * d] = o[d];
      __syncthreads();
      if ((w & 1) == 0 && i < c.rows) {
        m = fmaxf(m, part[w + 1][0]);
        l = 0.f;
#pragma unroll
        for (int d = 0; d < DL; ++d) o[d] = 0.f;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const float* p = part[w + q];
          const float f = p[0] == -kInf ? 0.f : fast_exp2(p[0] - m);
          l += f * p[1];
#pragma unroll
          for (int d = 0; d < DL; ++d) o[d] += f * p[2 + lane + 64 * d];
        }
        const int f = c.f0 + i;
        write_row<T, D>(a, c.row0 + f / a.group, c.head * a.group + f % a.group, m, l, o);
      }
      __syncthreads();
    }
  }
  if (a.zero_rest) {
    const int rows = static_cast<int>(a.b.rows);
    const int before = clamp_row(a.b.starts[0], rows), tail = clamp_row(a.b.starts[a.b.seqs], rows);
    const int64_t end = (before + static_cast<int64_t>(rows) - tail) * a.heads_q;
    const float none[DL] = {};
    for (int64_t x = blockIdx.x * 8 + w; x < end; x += gridDim.x * 8) {
      const int i = static_cast<int>(x / a.heads_q);
      write_row<T, D>(a, i < before ? i : i - before + tail, static_cast<int>(x % a.heads_q), -kInf, 0.f, none);
    }
  }
}

// ------------------------------------------------------------------ many rows a sequence
//
// Prompts: matrix products bound the work. Blocks of 128 flattened rows (row * group + head), 32 a wave, sweep tiles of 32
// keys that the workgroup stages in LDS, double-buffered; the products, the swizzled tiles, the softmax with a maximum that
// moves only when it must and the lazily read operands are the forward kernel's of flash_fwd.hip. The rows of a group lie
// side by side, so that a block spans few positions: at a group of 4, 32 of them, and one tile in 32 keys is cut by the diagonal.
//
// A tile's two halves of 16 keys lie in one page each. 16 bits: direct loads into LDS through a buffer resource per half,
// built from the half's page; keys that no row of the block sees are given an offset past the resource and read as zero.
// 4 bits: half of the threads fetch K's codes and scales, half V's, one load each, a tile ahead in registers, and widen them
// into the same LDS rows when the tile before is done with.
//
// Workgroups: a sequence's blocks come in slots starts * group / 128 + sequence onward (rounded down), which never overlap,
// so that the grid is known without the starts; a workgroup counts the sequences at or before its slot. Late blocks, which
// see the most keys, go first, in runs of four of alternating direction (the four shader engines of an XCD draw alike); an
// XCD works through few heads at a time, whose keys its L2 holds (SlotMap). A grid too small for the chip cuts each block's
// tiles into parts that paged_prompt_merge joins.
//
// The matrix pipe and the softmax's VALU share the clock that the part's power leaves: 2 x 4096 tokens, 32/8 heads of 128,
// 257-270 us on several cards (1020 to 1070 TFLOP/s; a library product of 8192^3 has 1200), 281 under a profiler, matrix pipe 48%
// busy, VALU 50%, 2.0 GHz. 8192 under a window of 1024: 148-158 us (820-870); of 35 tiles a block one in ten is cut or outside,
// and 4096 / 6144 / 8192 / 9216 / 12288 rows take 87 / 118 / 153 / 168 / 218 us: 16 us for 1000 more, 1050 TFLOP/s, and 30 us at
// the ends of the launch, where the chip fills and drains. 4 bits, 4 x 500 ragged rows over 7001: 148 us and 12 of joining
// (750), 33% busy: a tile's codes are widened between the products of two.

template <int D, int BITS>
struct ProCfg {
  static constexpr int BM = 128, BN = 32;
  static constexpr int ROWB = D * 2;
  static constexpr int CPR = D / 8;
  static constexpr int TILEB = BN * ROWB;
  static constexpr int KBUF = 0, VBUF = 2 * TILEB;
  static constexpr int LDS = 4 * TILEB;
  static constexpr int RPK = 1024 / ROWB;    // rows of a 1 KB direct load
  static constexpr int NDMA = BN / RPK / 4;  // loads of K, and of V, a wave and tile
  static constexpr int KS = D / 32;
  static constexpr int FB = D / 16;
  static constexpr int PF = 1;  // V operands in flight ahead of their product
  // K operands in flight: as many as the registers hold (4 bits, D = 128: the codes take theirs, and ten spill). 2 x 4096
  // tokens, 32/8 heads of 128, us: one of V and two of K 256, two and three 258, no more than two cards differ; 4 bits, one
  // and one 272, one and three 290, two and three 295
  static constexpr int KPF = BITS == 4 && D == 128 ? 1 : 2;
};

// The 16-byte slot of chunk c of a tile's row is c ^ this. Key rows are read as rows, 16 a load, value rows by the transposing
// 8-byte reads; both are conflict-free so, as in the forward kernel, whose layout this is.
template <int D>
__device__ __forceinline__ int key_swizzle(int row) {
  return D == 128 ? (row & 15) : (4 * (((row >> 1) ^ (row >> 3)) & 1) | 2 * ((row >> 2) & 1));
}
template <int D>
__device__ __forceinline__ int value_swizzle(int row) {
  return D == 128 ? 2 * (row & 7) : 2 * ((row & 3) ^ ((row >> 2) & 1));
}

constexpr float kTau = 8.0f;    // log2 of the growth of a row's maximum that is let pass
constexpr int kPartTiles = 8;   // no part of a block's keys is shorter, but the last

// A block's keys: tiles [0, sb) (the first tokens) and [wb, eb), cut into parts of `part` tiles.
struct BlockKeys {
  int sb, wb, tiles, part, parts;
  __device__ __forceinline__ int tile(int v) const { return v < sb ? v : v - sb + wb; }
};

__device__ __forceinline__ BlockKeys block_keys(const PagedAttn& a, int pos_lo, int pos_hi, int nsplit) {
  BlockKeys b;
  const int end = pos_hi + 1 < a.reach ? pos_hi + 1 : a.reach;
  const int eb = end > 0 ? (end + 31) / 32 : 0;
  const int lo = pos_lo - a.window + 1;
  b.wb = lo > 0 ? lo / 32 : 0;
  b.wb = b.wb < eb ? b.wb : eb;
  const int sink = a.sinks < end ? a.sinks : end;
  b.sb = sink > 0 ? (sink + 31) / 32 : 0;
  b.sb = b.sb < b.wb ? b.sb : b.wb;
  b.tiles = b.sb + eb - b.wb;
  b.part = (b.tiles + nsplit - 1) / nsplit;
  b.part = b.part > kPartTiles ? b.part : kPartTiles;
  b.parts = b.tiles > b.part ? (b.tiles + b.part - 1) / b.part : 1;
  return b;
}

// The sequence of a slot (seqs: the rows behind the last one; -1: none), the block's number in it, and the number of rows
// before the first sequence.
__device__ __forceinline__ int seq_of_slot(const PagedAttn& a, int slot, int& rb, int& before) {
  const int lane = threadIdx.x & 63, rows = static_cast<int>(a.b.rows);
  auto start = [&](int64_t i) { return a.b.seqs ? clamp_row(a.b.starts[i], rows) : 0; };
  auto base = [&](int64_t i) { return static_cast<int>(static_cast<int64_t>(start(i)) * a.group / 128 + i); };
  int n = 0;
  for (int64_t i = 0; i <= a.b.seqs; i += 64)
    n += __popcll(__builtin_amdgcn_ballot_w64(i + lane <= a.b.seqs && base(i + lane) <= slot));
  before = __builtin_amdgcn_readfirstlane(start(0));
  n = __builtin_amdgcn_readfirstlane(n) - 1;
  if (n >= 0) rb = slot - __builtin_amdgcn_readfirstlane(base(n));
  return n;
}

// Partial states of cut blocks: [nsplit][rows * heads_q] rows of o, then of (m in log2 units, l).
struct Parts {
  int nsplit;
  int64_t plane;  // rows * heads_q
  float* ws;
  template <int D>
  __device__ __forceinline__ float* o(int split, int64_t i) const {
    return ws + (split * plane + i) * D;
  }
  template <int D>
  __device__ __forceinline__ float* ml(int split, int64_t i) const {
    return ws + nsplit * plane * D + (split * plane + i) * 2;
  }
};

// Which workgroup takes which head and slot. Workgroups go round the eight XCDs; XCD x takes units x `units` and onward, a
// unit being every `shares`-th slot of a head (1 where the heads divide by eight), up to kHeadsRun of them at a time, the late
// slots of all of those first. Against whole heads one after the other, us, bf16: 2 x 4096 tokens, 12 heads of 64, 130 -> 88;
// 16 heads on one, 128 -> 104; 4 x 4096, 16 of 64, 192 -> 182; 2 x 4096, 32/8 of 128, 262 and 261. One unit at a time: 107,
// 104, 189, 266; eight: as three. Sequences in turn as well (two, four at a time): 80, 104, 174, 261, but 8 x 512 rows over
// 7001 keys 439 -> 478 and 459, their keys no longer in L2.
constexpr int kHeadsRun = 3;
struct SlotMap {
  int units, shares, unit_slots;
};

template <typename T, int D, int BITS, bool FAR>
__global__ __launch_bounds__(256, 3) void paged_prompt(PagedAttn a, Parts pt, SlotMap mp, int nslots) {
  using C = ProCfg<D, BITS>;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[C::LDS];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, G = lane >> 4, w = wave_id();
  const int R = a.group;

  // ---- workgroup -> part, head, slot
  int bid = blockIdx.x;
  const int split = scalar(bid % pt.nsplit);
  bid = scalar(bid / pt.nsplit);
  const int r = bid >> 3, per_run = kHeadsRun * mp.unit_slots;  // of this XCD's workgroups
  const int first = scalar(r / per_run) * kHeadsRun, in_run = scalar(r % per_run);
  const int n = mp.units - first < kHeadsRun ? mp.units - first : kHeadsRun;
  if (n <= 0) return;
  const int unit = (bid & 7) * mp.units + first + scalar(in_run % n);
  const int head = scalar(unit / mp.shares);
  int j = scalar(in_run / n);
  if ((j | 3) < mp.unit_slots && (j & 4)) j ^= 3;
  j = j * mp.shares + scalar(unit % mp.shares);
  if (j >= nslots) return;
  int rb = 0, before;
  const int seq = seq_of_slot(a, nslots - 1 - j, rb, before);
  if (before > 0 && a.zero_rest && split == 0) {  // rows before the first sequence, spread over the heads' slots
    const float none[D / 64] = {};
    const int64_t end = static_cast<int64_t>(before) * a.heads_q;
    for (int64_t x = (static_cast<int64_t>(head) * nslots + j) * 4 + w; x < end; x += a.c.heads * nslots * 4)
      write_row<T, D>(a, static_cast<int>(x / a.heads_q), static_cast<int>(x % a.heads_q), -kInf, 0.f, none);
  }
  if (seq < 0) return;
  const SeqPlan sp = uniform_plan<128>(a, seq);
  if (rb < 0 || rb >= sp.nb) return;

  // ---- the block's rows: lane row h of wave w is flattened row 128 rb + 32 w + 16 h + c
  const int f0 = rb * C::BM;
  const int fend = sp.n * R - f0 < C::BM ? sp.n * R : f0 + C::BM;  // rows x heads_q < 2^31
  const int pos_lo = scalar(sp.pos0 + f0 / R), pos_hi = scalar(sp.pos0 + (fend - 1) / R);
  BlockKeys bk = block_keys(a, pos_lo, pos_hi, pt.nsplit);
  bk.part = scalar(bk.part);
  bk.parts = scalar(bk.parts);
  if (split >= bk.parts) return;
  const int v0 = split * bk.part, v1 = v0 + bk.part < bk.tiles ? v0 + bk.part : bk.tiles;
  const int fw = f0 + 32 * w;
  const bool busy = fw < fend;  // this wave has rows
  const int wpos_hi = scalar(busy ? sp.pos0 + (fw + 31 < fend - 1 ? fw + 31 : fend - 1) / R : -1);
  int pos[2];
  u32x4 qreg[2][C::KS];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int f = fw + 16 * h + c;
    const bool live = f < fend;
    const int ff = live ? f : f0;
    pos[h] = live ? sp.pos0 + ff / R : -1;
    const uint16_t* qr = a.q + (sp.row0 + ff / R) * a.q_st + (head * R + ff % R) * a.q_sh;
#pragma unroll
    for (int ks = 0; ks < C::KS; ++ks) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(qr + ks * 32 + G * 8);
      qreg[h][ks] = live ? x : u32x4{0u, 0u, 0u, 0u};
    }
  }

  // ---- tiles: the pages of their two halves
  struct Tile {
    int key0, p[2];  // the pages as they stand in the table
  };
  const int32_t* trow = a.table + seq * a.b.ld_table;
  auto tile_at = [&](int v) {
    const int key0 = scalar(bk.tile(v) * 32), e0 = key0 >> a.shift, e1 = (key0 + 16) >> a.shift;
    return Tile{key0, {uniform_i32(trow + (e0 < a.last_entry ? e0 : a.last_entry)),
                       uniform_i32(trow + (e1 < a.last_entry ? e1 : a.last_entry))}};
  };
  auto gone = [&](const Tile& t, int at, int p) {  // no row of the block sees the key
    const int key = t.key0 + at;
    return !a.has(p) | (key > pos_hi) | (key >= a.reach) | ((key >= a.sinks) & (key <= pos_lo - a.window));
  };
  const int in_mask = (1 << a.shift) - 1;
  bool lost = false;  // a tile of a pair that every row should see whole lacks a page

  // ---- staging. A wave's part of a tile lies in one half, in one page: one buffer resource a pool with the page's place as
  // the scalar offset, or FAR, a resource a page; a lane's address is one offset that does not change.
  constexpr int ES = BITS == 16 ? 2 : 1;
  const uint32_t rst = static_cast<uint32_t>(a.c.sr) * ES, srst = static_cast<uint32_t>(a.c.ssr);
  const uint32_t whole_span = (a.pages - 1) * (static_cast<uint32_t>(a.c.sp) * ES) + in_mask * rst + D * BITS / 8;
  auto page_place = [&](int pg, int in, const char* pool, rsrc_t& r) {  // units of bytes
    if constexpr (FAR) {
      r = uniform_rsrc(pool + pool_at<BITS>(a.c, a.has(pg) ? pg : 0, in) * ES, 15 * rst + D * BITS / 8);
      return 0u;
    } else {
      return static_cast<uint32_t>(scalar((a.has(pg) ? pg : 0) * (static_cast<uint32_t>(a.c.sp) * ES) + in * rst));
    }
  };
  // 16 bits
  const char* const kpool = static_cast<const char*>(a.c.k) + head * a.c.sh * ES;
  const char* const vpool = static_cast<const char*>(a.c.v) + head * a.c.sh * ES;
  rsrc_t krs = uniform_rsrc(kpool, whole_span), vrs = uniform_rsrc(vpool, whole_span);
  const int lrow = lane / C::CPR, slot = lane % C::CPR;
  uint32_t dk[C::NDMA], dv[C::NDMA];
#pragma unroll
  for (int i = 0; i < C::NDMA; ++i) {
    const int at = (i * 4 + w) * C::RPK + lrow;
    dk[i] = lrow * rst + ((slot ^ key_swizzle<D>(at)) << 4);
    dv[i] = lrow * rst + ((slot ^ value_swizzle<D>(at)) << 4);
  }
  auto stage16 = [&](const Tile& t, int buf, bool cut) {
#pragma unroll
    for (int i = 0; i < C::NDMA; ++i) {
      const int blk = i * 4 + w, at0 = blk * C::RPK, h = at0 >> 4;  // its rows lie in one half
      const int pg = h ? t.p[1] : t.p[0], in = (t.key0 + at0) & in_mask;
      const uint32_t so = page_place(pg, in, kpool, krs);
      if constexpr (FAR) page_place(pg, in, vpool, vrs);
      uint32_t ok = dk[i], ov = dv[i];
      if (cut && gone(t, at0 + lrow, pg)) ok = ov = 0x7ffffff0u;  // past the resource: zeros
      dma16(krs, smem + C::KBUF + buf * C::TILEB + blk * 1024, ok, so);
      dma16(vrs, smem + C::VBUF + buf * C::TILEB + blk * 1024, ov, so);
    }
  };
  // 4 bits: waves 0 and 1 take K's halves, 2 and 3 V's; a lane a row and a chunk of D / 4 features
  typedef typename DecBlk<D, 4>::codes codes_t;
  codes_t codes{};
  uint32_t cbyte = 0;
  const bool isv = w >= 2;
  const int crow = 16 * (w & 1) + (lane >> 2), cch = lane & 3;
  const char* const cpool = isv ? vpool : kpool;
  const char* const spool = static_cast<const char*>(isv ? a.c.v_scale : a.c.k_scale) + head * a.c.ssh;
  rsrc_t crs = uniform_rsrc(cpool, whole_span);
  rsrc_t srs = uniform_rsrc(spool, (a.pages - 1) * static_cast<uint32_t>(a.c.ssp) + in_mask * srst + D / 32);
  const uint32_t coff = (lane >> 2) * rst + cch * (D / 8), soff = (lane >> 2) * srst + cch * (D / 4) / 32;
  auto fetch4 = [&](const Tile& t, bool cut) {
    const int pg = (w & 1) ? t.p[1] : t.p[0], in = (t.key0 + 16 * (w & 1)) & in_mask;
    const uint32_t so = page_place(pg, in, cpool, crs);
    uint32_t sso = 0;
    if constexpr (FAR)
      srs = uniform_rsrc(spool + scale_at(a.c, a.has(pg) ? pg : 0, in), 15 * srst + D / 32);
    else
      sso = scalar((a.has(pg) ? pg : 0) * static_cast<uint32_t>(a.c.ssp) + in * srst);
    codes = bload_codes<D>(crs, coff, so);
    cbyte = bload8(srs, soff, sso);
    if (cut && gone(t, crow, pg)) {
      codes = codes_t{};
      cbyte = 0;
    }
  };
  auto commit4 = [&](int buf) {
    unsigned char* dst = smem + (isv ? C::VBUF : C::KBUF) + buf * C::TILEB + crow * C::ROWB;
    const int swz = isv ? value_swizzle<D>(crow) : key_swizzle<D>(crow);
    const float cscale = e8m0(cbyte);
#pragma unroll
    for (int i = 0; i < C::KS; ++i)
      *reinterpret_cast<u32x4*>(dst + (((cch * C::KS + i) ^ swz) << 4)) = fp4_row8<T>(codes[i], cscale);
  };

  // ---- per-lane operand offsets
  int ka[C::KS];  // K row c, chunk 4 ks + G
#pragma unroll
  for (int ks = 0; ks < C::KS; ++ks) ka[ks] = c * C::ROWB + (((4 * ks + G) ^ key_swizzle<D>(c)) << 4);
  int va[C::FB];  // transposed V reads: row 4 G + k4 (+ 16), features 16 fb + 4 cc .. + 3
  {
    const int k4 = (lane >> 2) & 3, cc = lane & 3, r = 4 * G + k4;
#pragma unroll
    for (int fb = 0; fb < C::FB; ++fb)
      va[fb] = r * C::ROWB + (((2 * fb + (cc >> 1)) ^ value_swizzle<D>(r)) << 4) + ((cc & 1) << 3);
  }

  float mused[2] = {-kInf, -kInf}, lsum[2] = {0.f, 0.f};  // raw scores' reference, this lane's part of the sum
  f32x4 oacc[C::FB][2];
#pragma unroll
  for (int fb = 0; fb < C::FB; ++fb) oacc[fb][0] = oacc[fb][1] = f32x4{0.f, 0.f, 0.f, 0.f};

  auto vfrag = [&](const unsigned char* vt, int fb) {
    const u32x2 lo = ds_read_tr16(vt + va[fb]);
    const u32x2 hi = ds_read_tr16(vt + 16 * C::ROWB + va[fb]);
    return u32x4{lo.x, lo.y, hi.x, hi.y};
  };

  // buf: a constant where the tile is whole, so that every operand read is a lane's offset and an immediate
  auto tile = [&](auto buf, const Tile& t, auto cutc) __attribute__((always_inline)) {
    constexpr bool CUT = decltype(cutc)::value;
    const unsigned char* kt = smem + C::KBUF + buf * C::TILEB;
    const unsigned char* vt = smem + C::VBUF + buf * C::TILEB;
    f32x4 sacc[2][2];  // [key half][row half]: S^T[16 kb + 4 G + i][16 h + c]
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) sacc[kb][0] = sacc[kb][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto kfrag = [&](int n) { return *reinterpret_cast<const u32x4*>(kt + (n & 1) * 16 * C::ROWB + ka[n >> 1]); };
    u32x4 kf[C::KPF];
#pragma unroll
    for (int n = 0; n < C::KPF; ++n) kf[n] = kfrag(n);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int n = 0; n < 2 * C::KS; ++n) {
      const u32x4 kk = kf[n % C::KPF];
      if (n + C::KPF < 2 * C::KS) kf[n % C::KPF] = kfrag(n + C::KPF);
      const int ks = n >> 1, kb = n & 1;
      sacc[kb][0] = mfma16<T>(kk, qreg[0][ks], sacc[kb][0]);
      sacc[kb][1] = mfma16<T>(kk, qreg[1][ks], sacc[kb][1]);
    }
    u32x4 vf[C::PF];
#pragma unroll
    for (int n = 0; n < C::PF; ++n) vf[n] = vfrag(vt, n);
    __builtin_amdgcn_s_setprio(0);

    if constexpr (CUT) {  // key of accumulator (kb, i): key0 + 4 G + 16 kb + i
      const int kl = t.key0 + 4 * G;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int last = (pos[h] < a.reach ? pos[h] : a.reach - 1) - kl, first = pos[h] - a.window + 1 - kl;
        const int kept = a.sinks - kl;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          const int end = a.has(t.p[kb]) ? last : -1 - kMaxTokens;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int cc = 16 * kb + i;
            const bool seen = (cc <= end) & ((cc >= first) | (cc < kept));
            sacc[kb][h][i] = seen ? sacc[kb][h][i] : -kInf;
          }
        }
      }
    }
    u32x4 p[2];
    // what the exponentials refer to: 0 while a row's scores are all -inf, whose exponentials are then 0, not NaN
    auto ref = [&](int h) { return mused[h] == -kInf ? 0.f : mused[h]; };
    auto expo = [&](int h, float m) {
      const float mc = m * a.c2 - kLift<T>;
      float e[8];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = sacc[kb][h][i];
          if constexpr (!CUT)
            e[4 * kb + i] = fast_exp2(__builtin_fmaf(x, a.c2, -mc));
          else if constexpr (kLift<T> > 0.f)
            e[4 * kb + i] = fast_exp2(__builtin_fmaf(x - m, a.c2, kLift<T>));
          else
            e[4 * kb + i] = fast_exp2((x - m) * a.c2);
        }
      p[h] = u32x4{pack2<T>(e[0], e[1]), pack2<T>(e[2], e[3]), pack2<T>(e[4], e[5]), pack2<T>(e[6], e[7])};
      return ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
    };
    auto rowmax = [&](int h) {
      float m = -kInf;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i) m = fmaxf(m, sacc[kb][h][i]);
      return max4g(m);
    };
    auto rescale = [&](int h, float mnew) {
      const float alpha = mnew == mused[h] ? 1.f : fast_exp2((mused[h] - mnew) * a.c2);
      mused[h] = mnew;
      lsum[h] *= alpha;
#pragma unroll
      for (int fb = 0; fb < C::FB; ++fb) oacc[fb][h] *= alpha;
    };
    if constexpr (!CUT) {
      // a reference still at -inf makes these inf or NaN: over the limit
      float part0 = expo(0, mused[0]), part1 = expo(1, mused[1]);
      const float lim = static_cast<float>(1 << static_cast<int>(kTau + kLift<T>));
      if (__builtin_amdgcn_ballot_w64(!(part0 <= lim) || !(part1 <= lim)) != 0) {
        rescale(0, fmaxf(mused[0], rowmax(0)));
        rescale(1, fmaxf(mused[1], rowmax(1)));
        part0 = expo(0, ref(0));
        part1 = expo(1, ref(1));
      }
      lsum[0] += part0;
      lsum[1] += part1;
    } else {
      const float m0 = rowmax(0), m1 = rowmax(1);
      if (__builtin_amdgcn_ballot_w64((m0 - mused[0]) * a.c2 > kTau || (m1 - mused[1]) * a.c2 > kTau) != 0) {
        rescale(0, fmaxf(mused[0], m0));
        rescale(1, fmaxf(mused[1], m1));
      }
      lsum[0] += expo(0, ref(0));
      lsum[1] += expo(1, ref(1));
    }
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int fb = 0; fb < C::FB; ++fb) {
      const u32x4 vv = vf[fb % C::PF];
      if (fb + C::PF < C::FB) vf[fb % C::PF] = vfrag(vt, fb + C::PF);
      oacc[fb][0] = mfma16<T>(vv, p[0], oacc[fb][0]);
      oacc[fb][1] = mfma16<T>(vv, p[1], oacc[fb][1]);
    }
    __builtin_amdgcn_s_setprio(0);
  };

  // Tiles [c0, c1) are whole for every row of the block, as far as their pages are there; before them lie the first tokens
  // and the window's left edge, behind them the diagonal.
  int c0, c1;
  {
    const int edge = pos_hi - a.window + 1;
    const int first = edge > 0 ? (edge + 31) / 32 : 0, last = (pos_lo + 1 < a.reach ? pos_lo + 1 : a.reach) >> 5;
    c0 = bk.sb + (first > bk.wb ? first - bk.wb : 0);
    c1 = bk.sb + (last > bk.wb ? last - bk.wb : 0);
    if (c0 >= c1) c0 = c1 = bk.tiles;
    c0 = c0 < v0 ? v0 : (c0 > v1 ? v1 : c0);
    c1 = c1 < v0 ? v0 : (c1 > v1 ? v1 : c1);
  }
  if (v0 < v1) {
    auto bound = [&](int v) { return v < v1 ? v : v1 - 1; };
    // Whole tiles go in pairs; a last single one is computed, and therefore staged, with the cut ones: a half without a page
    // is zeros there, and a page of somebody else's, looked at afterwards (`lost`), in a pair alone.
    const int pairs = c0 + ((c1 - c0) & ~1);
    auto is_cut = [&](int v) { return v < c0 || v >= pairs; };
    Tile cur = tile_at(v0), next = tile_at(bound(v0 + 1));
    const int odd = c0 & 1;  // tile v lies in buffer (v ^ odd) & 1: the whole ones start in buffer 0
    if constexpr (BITS == 16) {
      stage16(cur, (v0 ^ odd) & 1, is_cut(v0));
    } else {
      fetch4(cur, is_cut(v0));
      commit4((v0 ^ odd) & 1);
    }
    auto one = [&](int v, auto buf, auto cutc) __attribute__((always_inline)) {
      if constexpr (BITS == 16) wait_vmcnt0();
      __syncthreads();
      const bool more = v + 1 < v1;
      if (more) {
        if constexpr (BITS == 16)
          stage16(next, buf ^ 1, is_cut(v + 1));
        else
          fetch4(next, is_cut(v + 1));
      }
      const Tile after = tile_at(bound(v + 2));
      if constexpr (decltype(cutc)::value) {
        if (cur.key0 <= wpos_hi) tile(buf, cur, cutc);
      } else {
        lost |= !(a.has(cur.p[0]) & a.has(cur.p[1]));
        if (busy) tile(buf, cur, cutc);
      }
      if constexpr (BITS == 4)
        if (more) commit4(buf ^ 1);
      cur = next;
      next = after;
    };
#pragma unroll 1
    for (int v = v0; v < v1;) {
#pragma unroll 1
      for (; v >= c0 && v < pairs; v += 2) {
        one(v, std::integral_constant<int, 0>{}, std::false_type{});
        one(v + 1, std::integral_constant<int, 1>{}, std::false_type{});
      }
      if (v < v1) {
        one(v, (v ^ odd) & 1, std::true_type{});
        ++v;
      }
    }
  }

  // ---- rows out: features 16 fb + 4 G + i of rows c, 16 + c
  unsigned again[2];  // rows (bit c) to do by themselves
  int fo = fw + c;
  asm volatile("" : "+v"(fo));  // rows and heads are found again here, not held through the sweep
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int f = fo + 16 * h;
    const bool live = f < fend;
    const int row = sp.row0 + f / R, hq = head * R + f % R;
    const float l = sum4g(lsum[h]);
    bool nan = l != l;
#pragma unroll
    for (int fb = 0; fb < C::FB; ++fb)
#pragma unroll
      for (int i = 0; i < 4; ++i) nan |= oacc[fb][h][i] != oacc[fb][h][i];
    unsigned long long b = __builtin_amdgcn_ballot_w64(nan && live);
    b |= b >> 32;
    again[h] = static_cast<unsigned>((b | (b >> 16)) & 0xffff);
    if (pos_lo == pos_hi) again[h] = 0;  // rows that see the same keys
    if (lost) again[h] = fw + 16 * h < fend ? (fend - fw - 16 * h < 16 ? (1u << (fend - fw - 16 * h)) - 1 : 0xffff) : 0;
    if (!live || (again[h] >> c & 1)) continue;
    const int64_t at = static_cast<int64_t>(row) * a.heads_q + hq;
    if (bk.parts > 1) {
      float* po = pt.o<D>(split, at) + 4 * G;
#pragma unroll
      for (int fb = 0; fb < C::FB; ++fb) *reinterpret_cast<f32x4*>(po + 16 * fb) = oacc[fb][h];
      if (G == 0) {
        float* ml = pt.ml<D>(split, at);
        ml[0] = mused[h] * a.c2 - kLift<T>;
        ml[1] = l;
      }
    } else {
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      uint16_t* out = a.o + row * a.o_st + hq * a.o_sh + 4 * G;
#pragma unroll
      for (int fb = 0; fb < C::FB; ++fb) {
        const f32x4 x = oacc[fb][h];
        *reinterpret_cast<u32x2*>(out + 16 * fb) = u32x2{pack2<T>(x[0] * inv, x[1] * inv), pack2<T>(x[2] * inv, x[3] * inv)};
      }
      if (G == 0 && a.lse) a.lse[at] = l == 0.f ? -kInf : (mused[h] * a.c2 - kLift<T> + __log2f(l)) * kLn2;
    }
  }
  // Rows at different positions share tiles: 0 times a value that only some of them see is NaN where it is an infinity or a
  // NaN. Such rows are done again, each by itself; all of them where a page is missing among tiles taken for whole.
#pragma unroll 1
  for (unsigned todo = again[0] | again[1] << 16; todo; todo &= todo - 1) {
    const int f = fw + __builtin_ctz(todo), tok = f / R, h = head * R + f % R;
    float m = -kInf, l = 0.f, o[D / 64] = {};
    const uint16_t* qr = a.q + (sp.row0 + tok) * a.q_st + h * a.q_sh;
    const int s1 = (v1 < bk.sb ? v1 : bk.sb) * 32;
    if (v0 < bk.sb) row_sweep<T, D, BITS>(a, seq, head, qr, sp.pos0 + tok, v0 * 32, s1, m, l, o);
    if (v1 > bk.sb)
      row_sweep<T, D, BITS>(a, seq, head, qr, sp.pos0 + tok, bk.tile(v0 > bk.sb ? v0 : bk.sb) * 32, bk.tile(v1 - 1) * 32 + 32,
                            m, l, o);
    if (bk.parts > 1) {
      const int64_t at = static_cast<int64_t>(sp.row0 + tok) * a.heads_q + h;
#pragma unroll
      for (int i = 0; i < D / 64; ++i) pt.o<D>(split, at)[lane + 64 * i] = o[i];
      if (lane == 0) {
        pt.ml<D>(split, at)[0] = m;
        pt.ml<D>(split, at)[1] = l;
      }
    } else {
      write_row<T, D>(a, sp.row0 + tok, h, m, l, o);
    }
  }
}

// Joins the parts of blocks that were cut. A lane takes four features, so that a wave has two heads of 128 at once (four of
// 64): a row's sequence and parts are looked up once for all of them, and their loads go together. Latency and bytes: 12 us
// for 42 MB of parts (4 x 500 ragged rows, two parts; one head a wave after another: 20).
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_prompt_merge(PagedAttn a, Parts pt) {
  constexpr int LPH = D / 4, HEADS = 256 / LPH;  // lanes a head, heads a workgroup
  const int row = blockIdx.x, h = blockIdx.y * HEADS + threadIdx.x / LPH, e = threadIdx.x % LPH * 4;
  const int seq = seq_of_row(a.b, row);
  if (seq >= a.b.seqs || h >= a.heads_q) return;
  const SeqPlan sp = uniform_plan<128>(a, seq);
  if (row < sp.row0 || row >= sp.row0 + sp.n) return;
  const int R = a.group;
  const int f0 = ((row - sp.row0) * R + h % R) / 128 * 128;
  const int fend = sp.n * R - f0 < 128 ? sp.n * R : f0 + 128;
  const int parts = block_keys(a, sp.pos0 + f0 / R, sp.pos0 + (fend - 1) / R, pt.nsplit).parts;
  if (parts <= 1) return;
  const int64_t at = static_cast<int64_t>(row) * a.heads_q + h;
  float m = -kInf, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < parts; ++s) {
    const float2 ml = *reinterpret_cast<const float2*>(pt.ml<D>(s, at));
    const f32x4 x = *reinterpret_cast<const f32x4*>(pt.o<D>(s, at) + e);
    const float mnew = fmaxf(m, ml.x);
    const float was = m == -kInf ? 0.f : fast_exp2(m - mnew), f = ml.x == -kInf ? 0.f : fast_exp2(ml.x - mnew);
    l = l * was + f * ml.y;
    o = o * was + x * f;
    m = mnew;
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  *reinterpret_cast<u32x2*>(a.o + row * a.o_st + h * a.o_sh + e) =
      u32x2{pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv)};
  if (e == 0 && a.lse) a.lse[at] = l == 0.f ? -kInf : (m + __log2f(l)) * kLn2;
}

}  // namespace
}  // namespace pdh

using namespace pdh;

namespace {

// The current device's compute units; asked for once a device (two runtime calls, 1 us, otherwise in every call).
int64_t compute_units() {
  static std::atomic<int> known[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  int n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    n = pdh_device_cus();
    n = n > 0 ? n : 256;
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// Rows a sequence and head that take the decode kernel: blocks of 16 flattened rows on average.
bool few_rows(const pdh_paged_batch& b, int64_t group) { return b.rows * group <= 16 * b.seqs; }

// Workgroups of the decode kernel: as many as run at once.
int decode_grid(const pdh_paged_cache& c) {
  return static_cast<int>(compute_units()) * (c.features == 128 ? (c.bits == 16 ? dec_wgs<128, 16>() : dec_wgs<128, 4>())
                                                                : (c.bits == 16 ? dec_wgs<64, 16>() : dec_wgs<64, 4>()));
}

// Parts that the prompt kernel cuts a block's keys into: as many as bring the grid nearest to two workgroups a compute unit,
// of at least 1024 keys of what the table can hold (the lengths are not known here; a block of fewer keys makes fewer
// parts). Measured, bf16, 32/8 heads of 128, us uncut / cut: 512 rows over 8192 keys 191 / 92, 128 over 8192 190 / 41, 4 x
// 500 ragged over 7001 188 / 150 (4 bits 212 / 165), 8 x 64 over 8192 197 / 100. Shorter parts lost: a prompt of 1024
// tokens in two 26% longer, of 2048 under a window of 1024 80%: those stay whole. At 128 over 8192 that is one workgroup a
// compute unit, 2.8 times the floor. Blocks are counted by rows alone; of sequences shorter than a block there are more, cut
// finer than the target. Counted by sequences too, us: 64 x 5 over 8192 418 -> 384 (4 bits 234 -> 245), 256 x 1 over 4096, 160/8
// heads, 819 -> 769, 24 x 8 over 8192 167 -> 160, but 64 x 1 ragged over 16000, 160/8, 636 -> 670, 24 x 20 over 4000, 12 heads of
// 64, 55 -> 62, 40 x 17 ragged over 9000, 16/4 of 64, 68 -> 77: neither is better throughout.
int prompt_splits(const pdh_paged_cache& c, const pdh_paged_batch& b, int64_t group, int64_t window, int64_t sinks) {
  const int64_t blocks = (b.rows * group / 128 + 1) * c.heads;
  int64_t keys = b.width * c.page_rows;
  if (window < keys && sinks < keys) keys = keys < window + sinks + 128 ? keys : window + sinks + 128;
  int64_t n = (4 * compute_units() + blocks) / (2 * blocks);
  n = n < keys / 1024 ? n : keys / 1024;
  return static_cast<int>(n < 1 ? 1 : (n < 32 ? n : 32));
}

}  // namespace

extern "C" size_t pdh_paged_attention_workspace(const pdh_paged_cache* cache, const pdh_paged_batch* batch,
                                                int64_t heads_q, int64_t window, int64_t sinks) {
  if (!cache || !batch || cache->heads < 1 || heads_q < cache->heads) return 0;
  if (few_rows(*batch, heads_q / cache->heads))
    return static_cast<size_t>(decode_grid(*cache)) * (sizeof(DecMeta) + 2 * 16 * (2 + cache->features) * sizeof(float));
  const int nsplit = prompt_splits(*cache, *batch, heads_q / cache->heads, window, sinks);
  if (nsplit == 1) return 0;
  return static_cast<size_t>(nsplit) * batch->rows * heads_q * (2 + cache->features) * sizeof(float);
}

extern "C" int pdh_paged_attention(const void* q, void* o, float* lse, int64_t heads_q, int64_t q_st, int64_t q_sh,
                                   int64_t o_st, int64_t o_sh, const pdh_paged_cache* cache,
                                   const pdh_paged_batch* batch, int64_t window, int64_t sinks, float scale,
                                   int zero_rest, void* ws, size_t ws_bytes, void* stream) {
  int shift = 0;
  const int rc = check_paged("pdh_paged_attention", cache, batch, &shift);
  if (rc) return rc;
  PDH_REQUIRE(heads_q >= 1 && heads_q <= 65535 && heads_q % cache->heads == 0, PDH_EINVAL,
              "pdh_paged_attention: heads_q must be a multiple of the cache's heads");
  PDH_REQUIRE(batch->rows * heads_q <= INT32_MAX, PDH_EINVAL, "pdh_paged_attention: rows * heads_q must be < 2^31");
  PDH_REQUIRE(window >= 1 && sinks >= 0, PDH_EINVAL, "pdh_paged_attention: window >= 1 and sinks >= 0");
  PDH_REQUIRE(std::isfinite(scale * kLog2e) && scale > 0.f, PDH_EINVAL, "pdh_paged_attention: scale must be finite and > 0");
  if (batch->rows == 0) return PDH_OK;
  PDH_REQUIRE(q && o && aligned16(q) && aligned16(o), PDH_EINVAL,
              "pdh_paged_attention: q and o must be 16-byte aligned");
  for (int64_t s : {q_st, q_sh, o_st, o_sh})
    PDH_REQUIRE(s >= 0 && s % 8 == 0, PDH_EINVAL, "pdh_paged_attention: strides must be multiples of 8 elements, >= 0");
  const Tokens out{o, batch->rows, heads_q, cache->features, o_st, o_sh}, in{q, batch->rows, heads_q, cache->features, q_st, q_sh};
  PDH_REQUIRE(out.spans().apart(), PDH_EINVAL, "pdh_paged_attention: o's rows overlap");
  PDH_REQUIRE(out.in_place_of(in) || out.spans().apart_from(in.spans()), PDH_EINVAL,
              "pdh_paged_attention: o overlaps q (it may be q, with q's strides)");
  PagedAttn a{static_cast<const uint16_t*>(q), static_cast<uint16_t*>(o), lse, q_st, q_sh, o_st, o_sh, *cache, *batch,
              static_cast<int>(heads_q), static_cast<int>(heads_q / cache->heads),
              static_cast<int>(window < kMaxTokens ? window : kMaxLength),  // of 2^30 and more: every position's whole past
              static_cast<int>(sinks < kMaxTokens ? sinks : kMaxTokens), shift, zero_rest != 0,
              static_cast<int>(batch->width << shift), scale * kLog2e,
              batch->width > 0 ? batch->table : batch->starts, static_cast<int>(batch->width > 0 ? batch->width - 1 : 0),
              static_cast<int>(cache->pages)};
  if (batch->width == 0) a.b.ld_table = 0;
  const size_t need = pdh_paged_attention_workspace(cache, batch, heads_q, window, sinks);
  PDH_REQUIRE(ws_bytes >= need && (need == 0 || (ws && aligned16(ws))), PDH_EINVAL,
              "pdh_paged_attention: workspace %zu bytes < required %zu, or not 16-byte aligned", ws_bytes, need);
  // what an offset from a head's first row has to reach, in bytes; to 2^31, so that 0x7ffffff0 lies past every resource and
  // no sum of two offsets wraps
  const int64_t pool = ((cache->pages - 1) * cache->sp + cache->page_rows * cache->sr) * (cache->bits == 16 ? 2 : 1);
  const int64_t scales = cache->bits == 4 ? (cache->pages - 1) * cache->ssp + cache->page_rows * cache->ssr : 0;
  const bool far = pool >= 0x7fff0000 || scales >= 0x7fff0000;
  const bool clear = clear_of_cache(out.spans(), *cache);
  if (few_rows(*batch, a.group)) {
    // The kernel sums up the work of all sequences, which starts that do not ascend may give all rows each, in 64 bits.
    const double most = static_cast<double>(batch->seqs) * static_cast<double>((batch->rows * a.group / 16 + 1) * cache->heads) *
                        static_cast<double>(a.reach / 32 + 1 + DecCfg<64, 16>::ITEM);
    PDH_REQUIRE(most < 4.6e18, PDH_EINVAL,
                "pdh_paged_attention: too many sequences, rows and tokens of the table: %g blocks of work, 2^62 at most", most);
    PDH_REQUIRE(clear, PDH_EINVAL, "pdh_paged_attention: o overlaps the cache");
    const unsigned n = static_cast<unsigned>(decode_grid(*cache));
    DecMeta* meta = static_cast<DecMeta*>(ws);
    float* states = reinterpret_cast<float*>(meta + n);
    by_kind(*cache, [&](auto t, auto d, auto bits) {
      using T = decltype(t);
      constexpr int D = decltype(d)::value;
      constexpr int B = decltype(bits)::value;
      if (!far)
        paged_decode<T, D, B, false><<<n, 256, 0, as_stream(stream)>>>(a, meta, states);
      else
        paged_decode<T, D, B, true><<<n, 256, 0, as_stream(stream)>>>(a, meta, states);
      paged_decode_merge<T, D><<<n, 512, 0, as_stream(stream)>>>(a, meta, states);
    });
    return check_launch("pdh_paged_attention (decode)");
  }
  const int nsplit = prompt_splits(*cache, *batch, a.group, window, sinks);
  const int64_t nslots = batch->rows * a.group / 128 + batch->seqs + 1;
  SlotMap mp{0, 1, 0};
  while (cache->heads * mp.shares % 8 != 0) mp.shares *= 2;
  mp.units = static_cast<int>(cache->heads * mp.shares / 8);
  mp.unit_slots = static_cast<int>((nslots + mp.shares - 1) / mp.shares);
  const int64_t blocks = int64_t{8} * mp.units * mp.unit_slots * nsplit;
  PDH_REQUIRE(blocks < (1 << 24), PDH_EINVAL, "pdh_paged_attention: too many rows and heads: %lld workgroups, at most 2^24 - 1",
              (long long)blocks);  // of 256 threads: a launch counts threads in 32 bits
  PDH_REQUIRE(clear, PDH_EINVAL, "pdh_paged_attention: o overlaps the cache");
  const Parts parts{nsplit, batch->rows * heads_q, static_cast<float*>(ws)};
  by_kind(*cache, [&](auto t, auto d, auto bits) {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    constexpr int B = decltype(bits)::value;
    const unsigned n = static_cast<unsigned>(blocks);
    if (!far)
      paged_prompt<T, D, B, false><<<n, 256, 0, as_stream(stream)>>>(a, parts, mp, static_cast<int>(nslots));
    else
      paged_prompt<T, D, B, true><<<n, 256, 0, as_stream(stream)>>>(a, parts, mp, static_cast<int>(nslots));
    if (nsplit > 1) {
      const dim3 grid(static_cast<unsigned>(batch->rows), static_cast<unsigned>((heads_q * D / 4 + 255) / 256));
      paged_prompt_merge<T, D><<<grid, 256, 0, as_stream(stream)>>>(a, parts);
    }
  });
  return check_launch("pdh_paged_attention (prompt)");
}
