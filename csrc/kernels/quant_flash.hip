// Attention of chunks of new tokens over the 8-bit cache (eia_quant.h), on v_mfma_f32_32x32x16_bf16.
//
// The queries of a sequence and the G heads of a kv head make rows (query, head), query first; a workgroup takes a block
// of them, 32 a wave, so that a tile of 64 keys and values is fetched once for the block whatever G is.  A wave holds its
// rows as columns: S^T[key, row] = K Q^T, then O^T[channel, row] += V^T P^T with P^T taken from the S^T accumulators as
// they lie (K rows enter with bits 2 and 3 of their number exchanged, so that an accumulator's elements are eight keys in
// a row).  A lane owns one row together with lane ^ 32.
//
// A tile comes from memory as codes, half the bytes of bf16, and is converted once on its way into LDS: a key's scale is
// the conversion's; values lie as sixteen tokens of a channel, whose scales differ, so each pair is converted twice and
// the halves are put together (24 instructions for 16 values).  Both are exact; the products run as with a bf16 cache, and as there
// weights are rounded to bf16, the operand's type (half a step, 2^-8 of each).  Their sum is that of the rounded pairs: one instruction adds both.
//
// The host lays the launch out (which rows, which tiles): blocks that would be the launch's tail are cut along the keys,
// their parts hand over fp32 sums and a second kernel puts them together.
//
// Bound by issue, and by power: 128 channels, of the 4300 cycles that two waves of a SIMD take for a tile each the matrix unit works in 2048 and
// the vector unit in some 2900 (exponentials, maxima, packing, conversion), LDS in 2300.  The halves of a workgroup take turns (by the
// clock, with its reads in the way: scores and conversion 1100 to 1300, outputs 670; codes asked for 400 to 600, weights 1400), 555 -> 544 us
// at 8192 tokens, 32 heads on 8; clocks fall from 2.2 to 2.0 GHz as the units fill.  1010 TFLOP/s of the causal half, where a plain bf16
// product of 8192^3 reaches 1281.  256 channels: 515 TFLOP/s (4096 tokens, 12 heads on 4), one wave a SIMD, whose products wait for its own
// vector work.  64: 680 (8192, 16 on 4), half the products for a score's seven vector instructions (scale and exponential, maximum, packing,
// sum, a share of the conversion).  By counters the vector and matrix units work in 57 and 28 % of the cycles with 64 channels, 45 and 43 with
// 128, 30 and 21 with 256.
// Measured and left: 64 rows a wave 732 us; the next tile's first product beside this one's exponentials 550 for 547; fp8 products
// with queries as two codes 527 for 542, but 4 us more in short launches and scores that lose their last bits.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "eia_flash.h"
#include "eia_quant.h"

namespace {

constexpr int FK = 64;               // keys of a tile

template <int D> struct Shape {
  // 128 channels: eight waves of 214 registers, two a SIMD, that share a tile's conversion (two workgroups of four waves: 8192 tokens,
  // 32 heads on 8, 558 -> 607 us).  256: four waves, one a SIMD (500 registers).  64: a tile is half the products, and a workgroup's
  // waves wait for one another at its end, so two workgroups of four waves take turns (one of eight -> two of four: 12 heads, four of
  // 900 behind 3000 80.9 -> 59.8 us, one of 2048 30.9 -> 24.7, 16 on 4, 4096 tokens 73.8 -> 62.6, 8192 200 -> 202).
  static constexpr int THREADS = D == 128 ? 512 : 256;
  static constexpr int WAVES = D == 64 ? 3 : D == 128 ? 2 : 1;    // a SIMD: what the registers are held to
  static constexpr int ROWS = THREADS / 64 * 32;
  static constexpr int KS = D + 8, VS = FK + 8;           // row strides in LDS: 16 bytes apart from a power of two
  static constexpr bool TURNS = THREADS == 512;           // halves of the workgroup multiply and weigh in turn
  static constexpr int NV = TURNS ? 3 : 2;                // value tiles in LDS
  static constexpr int LDS = 2 * FK * KS + NV * D * VS;
};

// A block of rows of a sequence (its first query, queries and keys): first row, first key, key tiles, place of a part's sums (-1:
// whole).  All that a workgroup would wait for one load after the other.
struct Item { int seq, row, lo, tiles, slot, qbeg, qlen, len; };
struct Merge { int row, slot, parts, qbeg, qlen, pad[3]; };

struct Chunk {
  const bf16_t* q;
  bf16_t* out;
  long q_stride, out_stride;
  const int* tables;
  int bt_stride, Hq, causal, window, chunk;
  float scale_log2;
  f32x4* po;                         // sums of a part as its lanes hold them [slot][kv head][wave][D / 8][64]
  float2* ml;                        // [slot][kv head][wave][32]
  int groups, longest;               // 16-key groups of a page; tokens that a row of the tables has pages for
  unsigned top;                      // the last page: tables are held to it
  unsigned magic;
};

EIA_DEV int swap_bits(int r) { return (r & ~12) | ((r & 4) << 1) | ((r & 8) >> 1); }

EIA_DEV int first_key(int qa, int window, int chunk) {
  int lo = 0;
  if (window > 0) lo = max(lo, qa - window + 1);
  if (chunk > 0 && qa > 0) lo = max(lo, qa / chunk * chunk);
  return lo;
}

// 32 channels of a row: lane half h holds channels 8 j + 4 h .. + 3; halves of pairs change places, for 16-byte stores.
EIA_DEV void put_row(bf16_t* op, const f32x16_t& o, float inv) {
  uint2 pk[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    pk[j] = make_uint2(__builtin_bit_cast(unsigned, flash_pack(o[4 * j] * inv, o[4 * j + 1] * inv)),
                       __builtin_bit_cast(unsigned, flash_pack(o[4 * j + 2] * inv, o[4 * j + 3] * inv)));
#pragma unroll
  for (int j = 0; j < 4; j += 2) {
    const auto x = __builtin_amdgcn_permlane32_swap(pk[j].x, pk[j + 1].x, false, false);
    const auto y = __builtin_amdgcn_permlane32_swap(pk[j].y, pk[j + 1].y, false, false);
    *reinterpret_cast<uint4*>(op + 8 * j) = make_uint4(x[0], y[0], x[1], y[1]);
  }
}

template <int D>
__global__ void __launch_bounds__(Shape<D>::THREADS, Shape<D>::WAVES)
quant_flash_kernel(Chunk a, QuantCache cache, const Item* __restrict__ items) {
  constexpr int NT = Shape<D>::THREADS, KS = Shape<D>::KS, VS = Shape<D>::VS, NV = Shape<D>::NV;
  constexpr bool TURNS = Shape<D>::TURNS;
  constexpr int PIECES = 4 * D;                            // 16-byte pieces of a tile's keys, and of its values
  constexpr int NP = PIECES / NT;
  static_assert(PIECES % NT == 0, "");
  __shared__ __align__(16) bf16_t lds[Shape<D>::LDS];
  bf16_t* const vlds = lds + 2 * FK * KS;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), r32 = lane & 31, h = lane >> 5;
  const Item it = items[blockIdx.y];
  const int kvh = blockIdx.x, Hkv = cache.Hkv, G = a.Hq / Hkv;
  const int qbeg = it.qbeg, qlen = it.qlen, L = min(it.len, a.longest), ctx = L - qlen;
  const int rows = qlen * G, row0 = it.row + 32 * w;
  const bool window = a.window > 0 || a.chunk > 0;
  const int row = min(row0 + r32, rows - 1), qi = row / G;
  const long tok = qbeg + qi;
  const int hq = kvh * G + row - qi * G;
  const int qa = ctx + qi, q_lo = first_key(qa, a.window, a.chunk);
  const int kmax = a.causal ? min(L - 1, qa) : L - 1;

  bf16x8 qf[D / 16];                                       // step t: channels 16 t + 8 h .. + 7
  {
    const bf16_t* qp = a.q + tok * a.q_stride + (long)hq * D + 8 * h;
#pragma unroll
    for (int t = 0; t < D / 16; ++t) qf[t] = *reinterpret_cast<const bf16x8*>(qp + 16 * t);
  }
  const bool live = row0 < rows;
  const int wq0 = min(row0, rows - 1) / G, wq1 = min(row0 + 31, rows - 1) / G;     // the wave's first and last query
  const int w_hi = !live ? 0 : a.causal ? min(L, ctx + wq1 + 1) : L;
  const int w_lo = first_key(ctx + wq0, a.window, a.chunk);

  const int* bt = a.tables + (long)it.seq * a.bt_stride;
  const int last = max(L - 1, 0) / QUANT_GROUP;
  auto piece = [&](int i) { return tid + NT * i; };
  // a wave's pieces of keys and of values lie in one group of 16 tokens, the same for both
  int page[NP], off[NP];
  auto look = [&](int tile) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int group = __builtin_amdgcn_readfirstlane(min((it.lo + FK * tile) / QUANT_GROUP + piece(i) / D, last));
      const int at = a.groups == 1 ? group : (int)__umulhi((unsigned)group, a.magic);
      page[i] = bt[at];
      off[i] = QUANT_GROUP * (a.groups == 1 ? 0 : group - at * a.groups);
    }
  };
  uint4 kst[NP], vst[NP], vsc[NP];
  unsigned ksc[NP];
  auto fetch = [&] {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int pg = quant_page(__builtin_amdgcn_readfirstlane(page[i]), a.top), id = piece(i);
      const int r = id / (D / 16) % QUANT_GROUP;
      kst[i] = *reinterpret_cast<const uint4*>(cache.key(pg, kvh, off[i] + r, D) + 16 * (id % (D / 16)));
      ksc[i] = *cache.kscale(pg, kvh, off[i] + r);
      vst[i] = *reinterpret_cast<const uint4*>(cache.values(pg, kvh, off[i], D) + 16 * (id % D));
      vsc[i] = *reinterpret_cast<const uint4*>(cache.vscale(pg, kvh, off[i]));
    }
  };
  // Before the conversion: codes of keys that are no number, values past the end (whatever lies there, nothing of it is kept).
  auto ready = [&](int tile) {
    const int kb = it.lo + FK * tile;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      if (ksc[i] == QUANT_POISON) {
        ksc[i] = 127;
        kst[i] = make_uint4(0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu);
      }
      if (kb + FK > L) {
        const int n = max(L - kb - QUANT_GROUP * (piece(i) / D), 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int left = min(max(n - 4 * j, 0), 4);
          const unsigned keep = left == 4 ? ~0u : (1u << (8 * left)) - 1;
          (&vst[i].x)[j] &= keep;
          (&vsc[i].x)[j] &= keep;
        }
      }
    }
  };
  // Half h of a thread's pieces, converted, into LDS.
  auto stash = [&](int kbuf, int vbuf, int i, int h) {
    bf16_t* kl = lds + kbuf * (FK * KS);
    bf16_t* vl = vlds + vbuf * (D * VS);
    const int id = piece(i);
    bf16_t *kp = kl + id / (D / 16) * KS + 16 * (id % (D / 16)) + 8 * h, *vp = vl + id % D * VS + QUANT_GROUP * (id / D) + 8 * h;
    *reinterpret_cast<bf16x8*>(kp) = quant_eight((&kst[i].x)[2 * h], (&kst[i].x)[2 * h + 1], quant_scale(ksc[i]));
    unsigned y[4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const unsigned word = (&vst[i].x)[2 * h + j], sb = __builtin_amdgcn_readfirstlane((&vsc[i].x)[2 * h + j]);
      float s[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) s[b] = quant_scale((sb >> (8 * b)) & 255u);
      y[2 * j] = (quant_pair<false>(word, s[0]) & 0xffffu) | (quant_pair<false>(word, s[1]) & 0xffff0000u);
      y[2 * j + 1] = (quant_pair<true>(word, s[2]) & 0xffffu) | (quant_pair<true>(word, s[3]) & 0xffff0000u);
    }
    *reinterpret_cast<uint4*>(vp) = make_uint4(y[0], y[1], y[2], y[3]);
  };
  auto stash_all = [&](int kbuf, int vbuf) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      stash(kbuf, vbuf, i, 0);
      stash(kbuf, vbuf, i, 1);
    }
  };

  f32x16_t o[D / 32];
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
  float m = -INFINITY, l = 0.f;
  const int krow = swap_bits(r32);

  auto ahead = [&](int t) {                                // behind the conversion of tile t + 1: tile t + 2 takes its registers
    if (t + 2 < it.tiles) {
      fetch();
      if (t + 3 < it.tiles) look(t + 3);
    }
  };
  f32x16_t sc[2];
  bf16x8 p[4];
  float sum[4];
  // scores of tile t; beside them tile t + 1 is converted.  Reads of LDS go four fragments ahead of the products
  auto scores = [&](int t, int vbuf) {
    const bf16_t* kf0 = lds + (t & 1) * (FK * KS) + krow * KS + 8 * h;
    bf16x8 kf[2][4];
    auto keys = [&](int b) {
#pragma unroll
      for (int x = 0; x < 4; ++x) kf[b & 1][x] = *reinterpret_cast<const bf16x8*>(kf0 + 32 * KS * (x & 1) + 16 * (2 * b + (x >> 1)));
    };
    keys(0);
#pragma unroll
    for (int b = 0; b < D / 32; ++b) {
      if (b + 1 < D / 32) keys(b + 1);
      __builtin_amdgcn_sched_barrier(0);
      if (b < 2 * NP) stash((t + 1) & 1, vbuf, b >> 1, b & 1);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int step = 2 * b + (x >> 1);
        sc[x & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[b & 1][x], qf[step], step == 0 ? f32x16_t{} : sc[x & 1], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // the tile's mask and maximum: element i of half sh is key kb + 32 sh + 16 (i / 8) + 8 h + i % 8
  float use;
  auto bound = [&](int kb) {
    const bool whole = !window && kb + FK <= L && (!a.causal || kb + FK - 1 <= ctx + wq0);
    mfma_settle(sc[0], sc[1]);
    if (!whole) {
      // seen: q_lo <= key <= kmax, as one unsigned comparison (a row that sees nothing compares with a far place)
      const unsigned lim = kmax >= q_lo ? (unsigned)(kmax - q_lo) : 0u;
      const int d0 = kmax >= q_lo ? kb + 8 * h - q_lo : 1 << 30;
#pragma unroll
      for (int sh = 0; sh < 2; ++sh)
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[sh][i] = (unsigned)(d0 + 32 * sh + 16 * (i >> 3) + (i & 7)) <= lim ? sc[sh][i] : -INFINITY;
    }
    float mx4[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      mx4[c] = sc[c >> 1][8 * (c & 1)];
#pragma unroll
      for (int j = 1; j < 8; ++j) mx4[c] = fmaxf(mx4[c], sc[c >> 1][8 * (c & 1) + j]);
    }
    const float mt = flash_pair_max(fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]))) * a.scale_log2;
    // the running maximum moves only where a tile exceeds it by more than 2^8: weights stay below 256, sums in fp32
    const bool grow = mt > m + FLASH_DEFER;
    if (__any(grow)) {
      const float now = grow ? mt : m, old = grow ? exp2f(m - now) : 1.f;
      m = now;
      l *= old;
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) o[dt] *= old;
    }
    use = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int c = 0; c < 4; ++c) sum[c] = 0.f;
  };
  auto weights = [&](int ks) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const f32x16_t& v = sc[ks >> 1];
      const int e = 8 * (ks & 1) + j;
      const bf16x2 y = flash_pack(__builtin_amdgcn_exp2f(fmaf(v[e], a.scale_log2, -use)), __builtin_amdgcn_exp2f(fmaf(v[e + 1], a.scale_log2, -use)));
      p[ks][j] = y[0];
      p[ks][j + 1] = y[1];
      sum[ks] = __builtin_amdgcn_fdot2_f32_bf16(y, bf16x2{(bf16_t)1.f, (bf16_t)1.f}, sum[ks], false);
    }
  };
  constexpr int VB = D / 32 < 4 ? D / 32 : 4, NB = D / 32 / VB;      // fragments of values read ahead, blocks of channels of them
  // the outputs of a tile; its weights formed beside the products, or there already
  auto outputs = [&](int vbuf, auto form) {
    const bf16_t* vf0 = vlds + vbuf * (D * VS) + r32 * VS + 8 * h;
    bf16x8 vf[2][VB];
    auto values = [&](int s) {                             // step s: channels of block s % NB, keys of s / NB
#pragma unroll
      for (int x = 0; x < VB; ++x) vf[s & 1][x] = *reinterpret_cast<const bf16x8*>(vf0 + 32 * VS * (VB * (s % NB) + x) + 16 * (s / NB));
    };
    values(0);
    __builtin_amdgcn_sched_barrier(0);
    if (form) weights(0);
#pragma unroll
    for (int s = 0; s < 4 * NB; ++s) {
      if (s + 1 < 4 * NB) {
        values(s + 1);
        if (form && (s + 1) % NB == 0) weights((s + 1) / NB);
      }
      if (!form) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int x = 0; x < VB; ++x)
        o[VB * (s % NB) + x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[s & 1][x], p[s / NB], o[VB * (s % NB) + x], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // Tile t is multiplied while tile t + 1 is converted, beside the first product, and tile t + 2 is on its way.
  if (it.tiles > 0) {
    look(0);
    fetch();
    look(min(1, it.tiles - 1));
    ready(0);
    stash_all(0, 0);
    if (it.tiles > 1) fetch();
    if (it.tiles > 2) look(2);
  }
  __syncthreads();
  // (behind the last tile the same registers go into a buffer that nobody reads)
  if constexpr (TURNS) {
    // Four waves, one on each SIMD, multiply (scores of tile t and the conversion beside it, outputs of tile t - 1) while the other
    // four form weights and ask for codes; then the halves change places.  Keys of tile t + 1 are stored while both halves may still read those of t, values
    // while t - 1 is read too: three places.  Every wave passes 2 T + 1 barriers.
    auto turn = [&] {
      __builtin_amdgcn_sched_barrier(0);
      __syncthreads();
      __builtin_amdgcn_sched_barrier(0);
    };
    const bool late = w >= NT / 128;
    if (late) turn();
    bool before = false;
    int was = NV - 1, at = 0;                                // places of the values of tiles t - 1 and t
    for (int t = 0; t < it.tiles; ++t) {
      const int kb = it.lo + FK * t, next = at == NV - 1 ? 0 : at + 1;
      const bool now = kb < w_hi && kb + FK > w_lo;        // (the same for the wave)
      ready(t + 1);
      __builtin_amdgcn_s_setprio(1);
      if (now) scores(t, next);
      else stash_all((t + 1) & 1, next);
      if (before) outputs(was, std::false_type{});
      __builtin_amdgcn_s_setprio(0);
      turn();
      ahead(t);
      if (now) {
        bound(kb);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) weights(ks);
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      }
      turn();
      before = now;
      was = at;
      at = next;
    }
    if (before) outputs(was, std::false_type{});
    if (!late) turn();
  } else {
    for (int t = 0; t < it.tiles; ++t) {
      const int kb = it.lo + FK * t;
      ready(t + 1);
      if (kb < w_hi && kb + FK > w_lo) {                   // (the same for the wave)
        __builtin_amdgcn_s_setprio(1);                     // products go before the other wave's vector work
        scores(t, (t + 1) & 1);
        __builtin_amdgcn_s_setprio(0);
        ahead(t);
        bound(kb);
        __builtin_amdgcn_s_setprio(2);
        outputs(t & 1, std::true_type{});
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        __builtin_amdgcn_s_setprio(0);
      } else {
        stash_all((t + 1) & 1, (t + 1) & 1);
        ahead(t);
      }
      __syncthreads();
    }
  }

#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) mfma_settle(o[dt]);
  const float lt = flash_pair_sum(l);
  if (it.slot >= 0) {
    if (!live) return;
    const long at = ((long)it.slot * Hkv + kvh) * (NT / 64) + w;
    f32x4* po = a.po + at * (D / 8 * 64) + lane;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int j = 0; j < 4; ++j) po[(4 * dt + j) * 64] = f32x4{o[dt][4 * j], o[dt][4 * j + 1], o[dt][4 * j + 2], o[dt][4 * j + 3]};
    if (h == 0) a.ml[at * 32 + r32] = make_float2(m, lt);
    return;
  }
  if (row0 + r32 >= rows) return;
  const float inv = lt != 0.f ? 1.f / lt : 0.f;
  bf16_t* op = a.out + tok * a.out_stride + (long)hq * D + 8 * h;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) put_row(op + 32 * dt, o[dt], inv);
}

// A workgroup puts the parts of one wave's 32 rows together, a wave 32 channels at a time.
template <int D>
__global__ void __launch_bounds__(256)
quant_flash_merge_kernel(Chunk a, int Hkv, const Merge* __restrict__ merges) {
  constexpr int W = Shape<D>::THREADS / 64;
  const Merge it = merges[blockIdx.z];
  const int kvh = blockIdx.x, w = blockIdx.y, lane = threadIdx.x & 63, r32 = lane & 31, h = lane >> 5, G = a.Hq / Hkv;
  const int qbeg = it.qbeg, rows = it.qlen * G, row0 = it.row + 32 * w;
  if (row0 >= rows) return;
  const long step = (long)Hkv * W, at = ((long)it.slot * Hkv + kvh) * W + w;
  const float2* ml = a.ml + at * 32 + r32;
  for (int dt = threadIdx.x >> 6; dt < D / 32; dt += 4) {
    const f32x4* po = a.po + at * (D / 8 * 64) + dt * 4 * 64 + lane;
    f32x16_t o;
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = 0.f;
    float m = -INFINITY, l = 0.f;
    for (int p0 = 0; p0 < it.parts; p0 += 4) {
      float2 x[4];
      f32x4 v[4][4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {                        // (a part past the last: the last one, weight 0)
        const long p = min(p0 + k, it.parts - 1) * step;
        x[k] = ml[p * 32];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[k][j] = po[p * (D / 8 * 64) + j * 64];
      }
      float mx = m;
#pragma unroll
      for (int k = 0; k < 4; ++k) mx = fmaxf(mx, x[k].x);
      const float use = mx == -INFINITY ? 0.f : mx, old = __builtin_amdgcn_exp2f(m - use);
      m = mx;
      l *= old;
      o *= old;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (p0 + k >= it.parts) break;
        const float c = __builtin_amdgcn_exp2f(x[k].x - use);
        l += c * x[k].y;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[4 * j + i] += c * v[k][j][i];
      }
    }
    const int row = row0 + r32, qi = row / G;
    if (row < rows)
      put_row(a.out + (long)(qbeg + qi) * a.out_stride + (long)(kvh * G + row - qi * G) * D + 8 * h + 32 * dt, o, l != 0.f ? 1.f / l : 0.f);
  }
}

}  // namespace

// Rows of a block (a workgroup's) at this head size; 0: not supported.
EIA_API int eia_quant_flash_rows(int D) {
  return D == 64 ? Shape<64>::ROWS : D == 128 ? Shape<128>::ROWS : D == 256 ? Shape<256>::ROWS : 0;
}

// items: n of {sequence, first row, first key, key tiles, slot or -1, first query, queries, keys}; merges: n_merge of {first row, first
// slot, parts, first query, queries, 3 unused}; ws: slots * Hkv * rows of a block * (D + 2) floats.
EIA_API int eia_quant_flash(const void* q, long q_stride, void* out, long out_stride, const void* k, const void* v, const void* ks,
                            const void* vs, long codes, long scales, int pages, const int* tables, int bt_stride, int width,
                            const int* items, int n, const int* merges, int n_merge, int slots, float* ws, float scale, int Hq, int Hkv,
                            int D, int bs, int causal, int window, int chunk, hipStream_t st) {
  if (n < 0 || n_merge < 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || bs <= 0 || bs % QUANT_GROUP || n > 65535 || n_merge > 65535 || pages < 0 || width < 0 ||
      (slots > 0 && !ws))
    return EIA_BAD_SHAPE;
  if (n == 0) return EIA_OK;
  const int groups = bs / QUANT_GROUP, block = eia_quant_flash_rows(D);
  if (!block) return EIA_UNSUPPORTED;
  const Chunk a{(const bf16_t*)q, (bf16_t*)out, q_stride, out_stride, tables, bt_stride, Hq, causal, window, chunk,
                scale * FLASH_LOG2E, reinterpret_cast<f32x4*>(ws), reinterpret_cast<float2*>(ws + (long)slots * Hkv * block * D), groups,
                pages ? (int)std::min<long>((long)width * bs, INT_MAX) : 0, pages ? pages - 1u : 0u,
                (unsigned)(((1ull << 32) + groups - 1) / groups)};
  const QuantCache c{(uint8_t*)k, (uint8_t*)v, (uint8_t*)ks, (uint8_t*)vs, codes, scales, Hkv, bs};
#define QF_GO(D)                                                                                                                 \
  do {                                                                                                                           \
    hipLaunchKernelGGL(quant_flash_kernel<D>, dim3(Hkv, n), dim3(Shape<D>::THREADS), 0, st, a, c, (const Item*)items);           \
    if (n_merge)                                                                                                                 \
      hipLaunchKernelGGL(quant_flash_merge_kernel<D>, dim3(Hkv, Shape<D>::THREADS / 64, n_merge), dim3(256), 0, st, a, Hkv, (const Merge*)merges); \
  } while (0)
  if (D == 64) QF_GO(64); else if (D == 128) QF_GO(128); else QF_GO(256);
#undef QF_GO
  EIA_LAUNCH_CHECK();
}
