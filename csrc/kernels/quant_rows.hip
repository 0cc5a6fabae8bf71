// Attention of a few queries a sequence over the 8-bit cache (eia_quant.h): decode, and chunks of few tokens.
//
// The queries of a sequence and the G heads of a kv head make rows (query, head), at most 16 NC of them, which are the
// columns of S^T = K Q^T and O^T = V^T P^T (v_mfma_f32_16x16x32_bf16).  A wave takes 64 keys at a time, straight from
// memory to registers: codes become bf16 operands there, exactly.
//   S^T, four tiles of 16 keys: row r of tile j is key 16 (r / 4) + 4 j + r % 4, so that lane (c, g) = (lane % 16, lane / 16)
//   ends up with the scores of keys 16 g .. 16 g + 15 of column c, and these, register by register, are the P^T operands
//   of two products whose V^T operand is the lane's 16 bytes of channel 16 dt + c: values[16 keys][channel][16].
// A key's scale goes into the conversion of its row; a value's, with which it would have to be multiplied byte by byte,
// into its weight.  Both are powers of two: exact.  The weight itself is rounded to bf16, the operand's type (half a step, 2^-8 of each, as with a
// bf16 cache); their sum is that of the fp32 weights, which the lane holds (a rounded one would have to be unpacked, and freed of the value's scale).
//
// A launch streams the cache once; its keys are cut into parts so that every row block, or a few long ones, load the
// whole chip.  All workgroups find the same cut from the sequences' lengths (plain sums of them: a few hundred numbers).
//
// A key and value are 2 (D + 1) bytes and 4 D operations for each of up to 16 NC columns: the cache's bytes bound long launches.
// 32 heads on 8 of 128, 32 rows of 8192 to 16384 keys 137 us, 6.1 TB/s (a kernel that only reads reaches 6.4); 65 of 1000 to 2000 42 us,
// 4.6 TB/s, parts that do not come out even.  Short launches are a chain of waits: lengths, table, keys, a unit or two a wave (2.4 us each
// with two column tiles), the waves' sums, the merge's launch: one row of 4000 keys 8.8 us in a graph.
// Four waves (RW) take every fourth unit and meet once at the end, or two every second, where there are more rows and heads than the chip holds
// workgroups of four (what these are for, short chains, is gone then).  32 heads on 8 of 128, us with four / two: 128 rows of 65 to 130 keys 14.5 /
// 12.3, of 250 to 500 30.6 / 27.4, of 1000 to 2000 79.2 / 72.8, 100 of 1000 to 2000 62.1 / 63.9; below that, 90 rows of 500 to 1000 33.2 /
// 38.1, one of 28749 on 4 heads 17.9 / 22.3.
// Tables wider than the longest row (a captured step's are as wide as the model is long): workgroups without a part search the cut and leave,
// which costs nothing to be seen; where no row is cut the merge is launched for nothing.  In a graph, tables as wide as the rows / 32768
// tokens: one row of 4000 9.1 / 9.0 us, 65 of 250 to 500 19.3 / 19.4, 65 of 65 to 130 9.2 / 11.7, 128 of 65 to 130 11.7 / 14.7.
// Meeting inside the kernel, the last part to arrive merging: one row 9.3 -> 9.9.
#include <algorithm>
#include <climits>

#include "eia_flash.h"
#include "eia_quant.h"

namespace {

constexpr int RU = 64;               // keys a wave takes at a time

struct Rows {
  const bf16_t* q;
  bf16_t* out;
  long q_stride, out_stride;
  const int *tables, *lens, *cu, *list;    // cu: first query of a sequence (nullptr: one each); list: the sequences (nullptr: all)
  int bt_stride, n, Hq, causal, window, chunk;
  float scale_log2;
  f32x4* po;                         // sums [part][kv head][column][D / 4]
  float2* ml;                        // maxima (log2), sums of weights [part][kv head][column]
  int2* info;                        // [sequence]: its first part and their number
  int per, least, share, groups;     // units a part (0: all over `share` workgroups, `least` at least); 16-key groups of a page
  int total, longest;                // parts that the launch has room for; tokens that a row of the tables has pages for
  unsigned top;                      // the last page: tables are held to it
  unsigned magic;                    // 2^32 / groups, rounded up
};

// Sums of the lanes up to each one, by lane moves in registers (over LDS they take the wave six round trips).
EIA_DEV int lanes_upto(int v) {
#define UPTO(move, rows) v += __builtin_amdgcn_update_dpp(0, v, move, rows, 0xf, true)
  UPTO(0x111, 0xf);                  // within sixteen lanes: from 1, 2, 4 and 8 below
  UPTO(0x112, 0xf);
  UPTO(0x114, 0xf);
  UPTO(0x118, 0xf);
  UPTO(0x142, 0xa);                  // the last of sixteen into the next sixteen (rows 1 and 3)
  UPTO(0x143, 0xc);                  // the last of 32 into the upper 32
#undef UPTO
  return v;
}

struct Span { int lo, units; };      // first unit, units

EIA_DEV Span rows_span(const Rows& r, int L, int qlen) {
  if (L <= 0 || qlen <= 0) return {0, 0};
  const int qa = max(L - qlen, 0);                          // position of the first query
  int lo = 0;
  if (r.window > 0) lo = max(lo, qa - r.window + 1);
  if (r.chunk > 0) lo = max(lo, qa / r.chunk * r.chunk);
  lo /= RU;
  return {lo, (L + RU - 1) / RU - lo};
}

// Units a part for so many in all: one round of the workgroups that run at a time, or two where that leaves parts of more than
// RLONG (their ends are apart then: 32 heads on 8, 32 rows of 8192 to 16384 keys in 512 parts 152 us, in 1024 144).
constexpr int RLONG = 48;
EIA_DEV int rows_per(const Rows& r, long units) {
  const int one = (int)((units + r.share - 1) / r.share), two = (one + 1) / 2;
  return max(r.least, min(one, max(two, RLONG)));
}

struct Part { int seq, L, q0, qlen, first, index, parts; Span span; };    // seq < 0: none

// The launch's part number y.  Every workgroup finds the same cut from the lengths, 64 sequences at a time: units a part so that
// the launch evens out over the workgroups that run at a time; a sequence has ceil(units / per) parts,
// one if it has no units, and parts are numbered through.
EIA_DEV Part rows_part(const Rows& r, int Hkv, int y) {
  const int lane = threadIdx.x & 63;
  auto length = [&](int i, int& s, int& L, int& q0, int& qlen) {
    s = i < r.n ? (r.list ? r.list[i] : i) : 0;
    L = i < r.n ? min(r.lens[s], r.longest) : 0;
    q0 = r.cu ? r.cu[s] : s;
    qlen = r.cu ? r.cu[s + 1] - q0 : 1;
  };
  int s, L, q0, qlen, per = r.per;
  length(lane, s, L, q0, qlen);
  if (per == 0) {
    int sum = 0;
    for (int i = lane; i < r.n; i += 64) {
      int s1 = s, L1 = L, q1 = q0, n1 = qlen;
      if (i != lane) length(i, s1, L1, q1, n1);
      sum += rows_span(r, L1, n1).units;
    }
    per = rows_per(r, (long)__builtin_amdgcn_readlane(lanes_upto(sum), 63) * Hkv);
  }
  const float inv = 1.f / (float)per;
  Part found{-1, 0, 0, 0, 0, 0, 0, {0, 0}};
  for (int i0 = 0, before = 0; i0 < r.n; i0 += 64) {
    if (i0) length(i0 + lane, s, L, q0, qlen);
    const Span span = rows_span(r, L, qlen);
    int parts = (int)((float)span.units * inv);             // ceil(units / per): a float's quotient may be one off
    parts += parts * per < span.units;
    parts -= (parts - 1) * per >= span.units;
    parts = i0 + lane < r.n ? max(parts, 1) : 0;
    const int upto = lanes_upto(parts);
    const int at = y - before;
    const unsigned long long mine = __ballot(at >= upto - parts && at < upto);
    if (mine) {
      const int from = __builtin_ctzll(mine);
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, from); };
      found = Part{of(s), of(L), of(q0), of(qlen), before + of(upto - parts), 0, of(parts), {of(span.lo), of(span.units)}};
      found.index = y - found.first;
      break;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return found;
}

EIA_DEV void put_rows(const Rows& r, int q0, int kvh, int G, int D, int col, int d, const f32x4& v, float sum) {
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  bf16x4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = f2bf(v[i] * inv);
  *reinterpret_cast<bf16x4*>(r.out + (long)(q0 + col / G) * r.out_stride + (long)(kvh * G + col % G) * D + d) = y;
}

template <int D, int NC, bool UNI, int RW>
__global__ void __launch_bounds__(64 * RW, D == 256 || NC == 2 ? 2 : D == 128 ? 3 : 4)
quant_rows_kernel(Rows r, QuantCache cache) {
  constexpr int KC = D / 64;         // 16-byte pieces of a key row a lane holds
  constexpr int DT = D / 16;
  constexpr bool AHEAD = D <= 128;   // keys are asked for a unit ahead; 256 channels: that costs the second workgroup on a CU
  __shared__ float sm[RW][16 * NC], sl[RW][16 * NC];
  __shared__ __align__(16) float so[RW][16 * NC][D + 4];      // (rows 16 bytes apart from a power of two)
  const int kvh = blockIdx.x, Hkv = cache.Hkv, G = r.Hq / Hkv;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
  const Part at = rows_part(r, Hkv, blockIdx.y);
  const int L = at.L, q0 = at.q0, qlen = at.qlen, nrow = min(qlen * G, 16 * NC), parts = at.parts;
  if (at.seq < 0) return;
  if (r.info && at.index == 0 && kvh == 0 && threadIdx.x == 0) r.info[at.seq] = make_int2(at.first, parts);
  if (nrow <= 0) return;
  const int* bt = r.tables + (long)at.seq * r.bt_stride;
  const Span span = at.span;
  const int each = (span.units + parts - 1) / parts;
  const int ub = span.lo + at.index * each, ue = min(ub + each, span.lo + span.units);

  // Q^T: step 2 i + h of the first product takes channels 64 i + 16 g + 8 h .. + 7 in lane group g.  In LDS: its registers
  // are worth a third workgroup on a CU.
  __shared__ bf16x8 qs[NC][2 * KC][64];
  int kmax[NC], klo[NC];
#pragma unroll
  for (int t = 0; t < NC; ++t) {
    const int row = min(16 * t + c, nrow - 1), qi = row / G;
    const bf16_t* qp = r.q + (long)(q0 + qi) * r.q_stride + (long)(kvh * G + row % G) * D + 16 * g;
#pragma unroll
    for (int i = 0; i < KC; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (((2 * i + h) & (RW - 1)) == w) qs[t][2 * i + h][lane] = *reinterpret_cast<const bf16x8*>(qp + 64 * i + 8 * h);
    const int qa = L - qlen + qi;
    kmax[t] = r.causal ? min(qa, L - 1) : L - 1;
    klo[t] = 0;
    if (r.window > 0) klo[t] = max(klo[t], qa - r.window + 1);
    if (r.chunk > 0) klo[t] = max(klo[t], qa / r.chunk * r.chunk);
  }
  const bool masks = r.window > 0 || r.chunk > 0 || qlen > 1;

  f32x4 o[NC][DT];
  float m[NC], l[NC];
#pragma unroll
  for (int t = 0; t < NC; ++t) {
    m[t] = -INFINITY, l[t] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[t][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const int last = max(L - 1, 0) / QUANT_GROUP;                   // the last group with a key: tables end there
  // 64 pages from one on, a lane each: a unit's page is a register's lane and no load in the loop
  auto index_of = [&](int group) { return r.groups == 1 ? group : (int)__umulhi((unsigned)group, r.magic); };
  int held = index_of(min(4 * (ub + w), last));
  int pages = ub + w < ue ? quant_page(bt[min(held + lane, index_of(last))], r.top) : 0;
  auto hold = [&](int group) {                              // (the same for the wave)
    const int at = index_of(group);
    if (at < held + 60) return;                             // (a unit lies in four pages at most)
    held = at;
    pages = quant_page(bt[min(held + lane, index_of(last))], r.top);
  };
  auto off_of = [&](int group) { return QUANT_GROUP * (group - index_of(group) * r.groups); };
  // Where a unit's keys and values lie: page and first token in it, one pair for a unit that one page holds (UNI), else a
  // pair for the lane's keys and one for its values.
  struct Place { int pk, ok, pv, ov; };
  auto look = [&](int u) {
    Place x;
    hold(__builtin_amdgcn_readfirstlane(min(4 * u, last)));
    if constexpr (UNI) {
      const int at = __builtin_amdgcn_readfirstlane(4 * u);
      x.ok = x.ov = off_of(at);
      x.pk = x.pv = __builtin_amdgcn_readlane(pages, index_of(at) - held);
    } else {
      const int gk = min(4 * u + (c >> 2), last), gv = min(4 * u + g, last);
      x = Place{__shfl(pages, index_of(gk) - held, 64), off_of(gk), __shfl(pages, index_of(gv) - held, 64), off_of(gv)};
    }
    return x;
  };
  // codes are read once, by one workgroup: past the caches (8 kv heads, 32 rows of 8192 to 16384 keys 164 -> 151 us, 64 of 2048 52.4 -> 47.3)
  uint4 k[4][KC], ks, v[DT], vs;
  auto load_keys = [&](const Place& x) {
    const int page = UNI ? __builtin_amdgcn_readfirstlane(x.pk) : x.pk;
    const uint8_t* p = cache.key(page, kvh, x.ok, D) + ((UNI ? 16 * (c >> 2) : 0) + (c & 3)) * D + 16 * g;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < KC; ++i) k[j][i] = quant_load<true>(p + 4 * j * D + 64 * i);
    ks = *reinterpret_cast<const uint4*>(cache.kscale(page, kvh, x.ok) + (UNI ? 16 * (c >> 2) : 0));
  };
  auto load_values = [&](const Place& x) {
    const int page = UNI ? __builtin_amdgcn_readfirstlane(x.pv) : x.pv;
    const uint8_t* p = cache.values(page, kvh, x.ov, D) + (UNI ? 16 * g * D : 0) + 16 * c;
    vs = *reinterpret_cast<const uint4*>(cache.vscale(page, kvh, x.ov) + (UNI ? 16 * g : 0));
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) v[dt] = quant_load<true>(p + 256 * dt);
  };
  Place next;
  auto compute = [&](int u, bool more) {
    // scales of this lane's four key rows
    unsigned kb[4], worst = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      kb[j] = ((&ks.x)[j] >> (8 * (c & 3))) & 255u;
      worst = max(worst, kb[j]);
    }
    if (__any(worst == QUANT_POISON)) {                     // a token that is no number: every code of its key becomes one
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (kb[j] == QUANT_POISON) {
          kb[j] = 127;
#pragma unroll
          for (int i = 0; i < KC; ++i) k[j][i] = make_uint4(0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu);
        }
    }
    if (RU * (u + 1) > L) {                                 // keys past the end: whatever lies there, nothing of it is kept
      const int n = min(max(L - RU * u - 16 * g, 0), 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int left = min(max(n - 4 * j, 0), 4);
        const unsigned keep = left == 4 ? ~0u : (1u << (8 * left)) - 1;
        (&vs.x)[j] &= keep;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) (&v[dt].x)[j] &= keep;
      }
    }
    f32x4 sc[NC][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float ksc = quant_scale(kb[j]);
#pragma unroll
      for (int t = 0; t < NC; ++t) sc[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        const bf16x8 a = quant_eight(k[j][i].x, k[j][i].y, ksc), b = quant_eight(k[j][i].z, k[j][i].w, ksc);
#pragma unroll
        for (int t = 0; t < NC; ++t) {
          sc[t][j] = mfma_bf16_k32(a, qs[t][2 * i][lane], sc[t][j]);
          sc[t][j] = mfma_bf16_k32(b, qs[t][2 * i + 1][lane], sc[t][j]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    // the next unit's keys take these registers; its values those of this unit's, below
    __builtin_amdgcn_sched_barrier(0);
    if (AHEAD && more) load_keys(next);
    __builtin_amdgcn_sched_barrier(0);
    bf16x8 p[NC][2];
    const bool part_seen = masks || RU * (u + 1) > L;
#pragma unroll
    for (int t = 0; t < NC; ++t) {
      mfma_settle(sc[t]);
      if (part_seen) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = RU * u + 16 * g + 4 * j + i;
            if (key > kmax[t] || key < klo[t]) sc[t][j][i] = -INFINITY;
          }
      }
      float mx = sc[t][0][0];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, sc[t][j][i]);
      const float now = fmaxf(m[t], column_max(mx) * r.scale_log2), use = now == -INFINITY ? 0.f : now;
      const float old = __builtin_amdgcn_exp2f(m[t] - use);
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = __builtin_amdgcn_exp2f(fmaf(sc[t][j][i], r.scale_log2, -use));
          sum += e;
          p[t][j >> 1][4 * (j & 1) + i] = f2bf(e * quant_scale(((&vs.x)[j] >> (8 * i)) & 255u));
        }
      l[t] = fmaf(l[t], old, sum);
      m[t] = now;
      if (!__all(old == 1.f)) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[t][dt] *= old;
      }
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const bf16x8 a = quant_eight(v[dt].x, v[dt].y, 1.f), b = quant_eight(v[dt].z, v[dt].w, 1.f);
#pragma unroll
      for (int t = 0; t < NC; ++t) {
        o[t][dt] = mfma_bf16_k32(a, p[t][0], o[t][dt]);
        o[t][dt] = mfma_bf16_k32(b, p[t][1], o[t][dt]);
      }
      if (dt & 1) __builtin_amdgcn_sched_barrier(0);
    }
  };
  int u = ub + w;
  if (u < ue) {
    next = look(u);
    load_keys(next);
    load_values(next);
    if (u + RW < ue) next = look(u + RW);
  }
  __syncthreads();
  if (u < ue) {
    for (;;) {
      const bool more = u + RW < ue;
      compute(u, more);
      if (!more) break;
      __builtin_amdgcn_sched_barrier(0);
      if (!AHEAD) load_keys(next);
      load_values(next);
      u += RW;
      if (u + RW < ue) next = look(u + RW);
    }
  }

#pragma unroll
  for (int t = 0; t < NC; ++t) {
    const float lt = column_sum(l[t]);
    if (g == 0) sm[w][16 * t + c] = m[t], sl[w][16 * t + c] = lt;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) mfma_settle(o[t][dt]);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(&so[w][16 * t + c][16 * dt + 4 * g]) = o[t][dt];
  }
  __syncthreads();
  const long base = ((long)blockIdx.y * Hkv + kvh) * (16 * NC);
  for (int id = threadIdx.x; id < nrow * (D / 4); id += 64 * RW) {
    const int col = id / (D / 4), d = id % (D / 4) * 4;
    float mx = sm[0][col];
#pragma unroll
    for (int k = 1; k < RW; ++k) mx = fmaxf(mx, sm[k][col]);
    const float use = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f;
    f32x4 v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < RW; ++k) {
      const float f = __builtin_amdgcn_exp2f(sm[k][col] - use);
      sum += sl[k][col] * f;
      const f32x4 y = *reinterpret_cast<const f32x4*>(&so[k][col][d]);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += y[i] * f;
    }
    if (parts > 1) {
      r.po[(base + col) * (D / 4) + d / 4] = v;
      if (d == 0) r.ml[base + col] = make_float2(mx, sum);
    } else {
      put_rows(r, q0, kvh, G, D, col, d, v, sum);
    }
  }
}

// The parts of a sequence's rows put together: one row a workgroup, D / 4 lanes across it, 1024 / D parts side by side, four of a
// thread's at a time.
template <int D, int NC>
__global__ void __launch_bounds__(256)
quant_rows_merge_kernel(Rows r, int Hkv) {
  constexpr int LANES = D / 4, PG = 256 / LANES;
  __shared__ float sm[PG], sl[PG];
  __shared__ f32x4 so[PG][LANES];
  const int kvh = blockIdx.x, G = r.Hq / Hkv, col = blockIdx.z, pg = threadIdx.x / LANES, d = threadIdx.x % LANES;
  const int s = r.list ? r.list[blockIdx.y] : blockIdx.y;
  const int2 at = r.info[s];                                // (of a sequence whose parts had no room in the launch: anything)
  if (at.x < 0 || at.x >= r.total) return;
  const int q0 = r.cu ? r.cu[s] : s, qlen = r.cu ? r.cu[s + 1] - q0 : 1, parts = min(at.y, r.total - at.x);
  if (parts <= 1 || col >= qlen * G) return;
  const long base = ((long)at.x * Hkv + kvh) * (16 * NC) + col, step = (long)Hkv * (16 * NC);
  float m = -INFINITY, l = 0.f;
  f32x4 v{0.f, 0.f, 0.f, 0.f};
  for (int p0 = pg; p0 < parts; p0 += 4 * PG) {
    float2 x[4];
    f32x4 y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {                           // (a part past the last: the last one, weight 0)
      const long p = base + min(p0 + k * PG, parts - 1) * step;
      x[k] = r.ml[p];
      y[k] = r.po[p * LANES + d];
    }
    float mx = m;
#pragma unroll
    for (int k = 0; k < 4; ++k) mx = fmaxf(mx, x[k].x);
    const float use = mx == -INFINITY ? 0.f : mx, old = __builtin_amdgcn_exp2f(m - use);
    m = mx;
    l *= old;
    v *= old;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (p0 + k * PG >= parts) break;
      const float f = __builtin_amdgcn_exp2f(x[k].x - use);
      l += x[k].y * f;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += y[k][i] * f;
    }
  }
  so[pg][d] = v;
  if (d == 0) sm[pg] = m, sl[pg] = l;
  __syncthreads();
  if (pg) return;
  m = sm[0];
#pragma unroll
  for (int k = 1; k < PG; ++k) m = fmaxf(m, sm[k]);
  const float use = m == -INFINITY ? 0.f : m;
  l = 0.f;
  v = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < PG; ++k) {
    const float f = __builtin_amdgcn_exp2f(sm[k] - use);
    l += sl[k] * f;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += so[k][d][i] * f;
  }
  put_rows(r, q0, kvh, G, D, col, 4 * d, v, l);
}

}  // namespace

// n sequences (list names them, or the first n; list entries and `sequences` bound them), each with at most 16 * tiles rows (query,
// head of a kv head); per: units of 64 keys a part (0: all over `share` workgroups, `least` at least); waves of a workgroup: 4, or 2 (one tile, D <= 128); parts: that many at most, n alone if no sequence
// is cut; ws (parts > n): parts * Hkv * 16 * tiles * (D + 2) floats, then 2 ints for every sequence.
EIA_API int eia_quant_rows(const void* q, long q_stride, void* out, long out_stride, const void* k, const void* v, const void* ks,
                           const void* vs, long codes, long scales, int pages, const int* tables, int bt_stride, int width, const int* lens, const int* cu,
                           const int* list, int n, float scale, int Hq, int Hkv, int D, int bs, int causal, int window, int chunk,
                           int tiles, int parts, int per, int least, int share, int waves, float* ws, hipStream_t st) {
  if (n < 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || bs <= 0 || bs % QUANT_GROUP || parts < n || pages < 0 || width < 0 || (parts > n && !ws) || parts > 65535 ||
      per < 0 || least < 1 || share < 1 || (waves != 4 && (waves != 2 || tiles > 1 || D > 128)) || tiles < 1)
    return EIA_BAD_SHAPE;
  if (n == 0) return EIA_OK;
  const int groups = bs / QUANT_GROUP;
  const long rows = (long)parts * Hkv * 16 * tiles;
  Rows r{(const bf16_t*)q, (bf16_t*)out, q_stride, out_stride, tables, lens, cu, list, bt_stride, n, Hq, causal, window, chunk,
         scale * FLASH_LOG2E, nullptr, nullptr, nullptr, per, least, share, groups, parts,
         pages ? (int)std::min<long>((long)width * bs, INT_MAX) : 0, pages ? pages - 1u : 0u,
         (unsigned)(((1ull << 32) + groups - 1) / groups)};
  if (parts > n) {
    r.po = reinterpret_cast<f32x4*>(ws);
    r.ml = reinterpret_cast<float2*>(ws + rows * D);
    r.info = reinterpret_cast<int2*>(ws + rows * (D + 2));
  } else {
    r.per = 1 << 30;
  }
  const QuantCache c{(uint8_t*)k, (uint8_t*)v, (uint8_t*)ks, (uint8_t*)vs, codes, scales, Hkv, bs};
#define RW_ROWS(D, NC, W)                                                                                                     \
  do {                                                                                                                        \
    if (bs % RU == 0) hipLaunchKernelGGL((quant_rows_kernel<D, NC, true, W>), dim3(Hkv, parts), dim3(64 * W), 0, st, r, c);   \
    else hipLaunchKernelGGL((quant_rows_kernel<D, NC, false, W>), dim3(Hkv, parts), dim3(64 * W), 0, st, r, c);               \
  } while (0)
#define RW_GO(D, NC)                                                                                                      \
  do {                                                                                                                    \
    if constexpr (NC == 1 && D <= 128) {                                                                                  \
      if (waves == 2) RW_ROWS(D, NC, 2); else RW_ROWS(D, NC, 4);                                                          \
    } else {                                                                                                              \
      RW_ROWS(D, NC, 4);                                                                                                  \
    }                                                                                                                     \
    if (parts > n)                                                                                                        \
      hipLaunchKernelGGL((quant_rows_merge_kernel<D, NC>), dim3(Hkv, n, cu ? 16 * NC : Hq / Hkv), dim3(256), 0, st, r, Hkv); \
  } while (0)
  if (tiles > (D == 256 ? 1 : 2)) return EIA_UNSUPPORTED;   // (more do not fit the registers)
  switch (D) {
    case 64: if (tiles == 1) RW_GO(64, 1); else RW_GO(64, 2); break;
    case 128: if (tiles == 1) RW_GO(128, 1); else RW_GO(128, 2); break;
    case 256: RW_GO(256, 1); break;
    default: return EIA_UNSUPPORTED;
  }
#undef RW_GO
#undef RW_ROWS
  EIA_LAUNCH_CHECK();
}
