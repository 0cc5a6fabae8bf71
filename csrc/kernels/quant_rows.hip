// Attention of a few queries a sequence over the 8-bit cache (eia_quant.h): decode, and chunks of few tokens.
//
// The queries of a sequence and the G heads of a kv head make rows (query, head), at most 16 NC of them, which are the
// columns of S^T = K Q^T and O^T = V^T P^T (v_mfma_f32_16x16x32_bf16).  A wave takes 64 keys at a time, straight from
// memory to registers: codes become bf16 operands there, exactly.
//   S^T, four tiles of 16 keys: row r of tile j is key 16 (r / 4) + 4 j + r % 4, so that lane (c, g) = (lane % 16, lane / 16)
//   ends up with the scores of keys 16 g .. 16 g + 15 of column c, and these, register by register, are the P^T operands
//   of two products whose V^T operand is the lane's 16 bytes of channel 16 dt + c: values[16 keys][channel][16].
// A key's scale goes into the conversion of its row; a value's, with which it would have to be multiplied byte by byte,
// into its weight.  Both are powers of two: exact.
//
// A launch streams the cache once; its keys are cut into parts so that every row block, or a few long ones, load the
// whole chip.  All workgroups find the same cut from the sequences' lengths (plain sums of them: a few hundred numbers).
#include "eia_flash.h"
#include "eia_quant.h"

namespace {

constexpr int RU = 64;               // keys a wave takes at a time
constexpr int RW = 4;                // waves of a workgroup

struct Rows {
  const bf16_t* q;
  bf16_t* out;
  long q_stride, out_stride;
  const int *tables, *lens, *cu, *list;    // cu: first query of a sequence (nullptr: one each); list: the sequences (nullptr: all)
  int bt_stride, n, Hq, causal, window, chunk;
  float scale_log2;
  float *po;                         // sums [sequence][kv head][part][column][D]
  float2* ml;                        // maxima (log2), sums of weights [sequence][kv head][part][column]
  int most, per, slots, groups;      // parts at most; units a part (0: from all lengths and the workgroups that run at a time); 16-key groups of a page
  unsigned magic;                    // 2^32 / groups, rounded up
};

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

// Units a part: what evens the launch out over the workgroups that run at a time, four (one a wave) at least.
EIA_DEV int rows_per(const Rows& r, int Hkv) {
  if (r.per > 0) return r.per;
  int sum = 0;
  for (int i = threadIdx.x & 63; i < r.n; i += 64) {
    const int s = r.list ? r.list[i] : i;
    sum += rows_span(r, r.lens[s], r.cu ? r.cu[s + 1] - r.cu[s] : 1).units;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  return max(RW, (int)(((long)sum * Hkv + r.slots - 1) / r.slots));
}
EIA_DEV int rows_parts(const Rows& r, int units, int per) { return max(1, min((units + per - 1) / per, r.most)); }

template <int D, int NC, bool UNI>
__global__ void __launch_bounds__(64 * RW, D <= 128 ? 2 : 1)
quant_rows_kernel(Rows r, QuantCache cache) {
  constexpr int KC = D / 64;         // 16-byte pieces of a key row a lane holds
  constexpr int DT = D / 16;
  __shared__ float sm[RW][16 * NC], sl[RW][16 * NC];
  __shared__ __align__(16) float so[RW][D][16 * NC + 1];
  const int kvh = blockIdx.x, part = blockIdx.z, Hkv = cache.Hkv, G = r.Hq / Hkv;
  const int s = r.list ? r.list[blockIdx.y] : blockIdx.y;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
  const int L = r.lens[s], q0 = r.cu ? r.cu[s] : s, qlen = r.cu ? r.cu[s + 1] - q0 : 1, nrow = min(qlen * G, 16 * NC);
  const int* bt = r.tables + (long)s * r.bt_stride;
  const Span span = rows_span(r, L, qlen);
  const int parts = rows_parts(r, span.units, rows_per(r, Hkv));
  if (part >= parts || nrow <= 0) return;
  const int each = (span.units + parts - 1) / parts;
  const int ub = span.lo + part * each, ue = min(ub + each, span.lo + span.units);

  // Q^T: step 2 i + h of the first product takes channels 64 i + 16 g + 8 h .. + 7 in lane group g
  bf16x8 qf[NC][2 * KC];
  int kmax[NC], klo[NC];
#pragma unroll
  for (int t = 0; t < NC; ++t) {
    const int row = min(16 * t + c, nrow - 1), qi = row / G;
    const bf16_t* qp = r.q + (long)(q0 + qi) * r.q_stride + (long)(kvh * G + row % G) * D + 16 * g;
#pragma unroll
    for (int i = 0; i < KC; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) qf[t][2 * i + h] = *reinterpret_cast<const bf16x8*>(qp + 64 * i + 8 * h);
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

  const int last = (L - 1) / QUANT_GROUP;                   // the last group with a key: tables end there
  auto page_of = [&](int group) { return bt[r.groups == 1 ? group : (int)__umulhi((unsigned)group, r.magic)]; };
  auto off_of = [&](int group) { return QUANT_GROUP * (r.groups == 1 ? 0 : group - (int)__umulhi((unsigned)group, r.magic) * r.groups); };
  struct Unit {
    uint4 k[4][KC], v[DT], ks, vs;
  };
  auto load = [&](Unit& x, int u) {
    const uint8_t *kp, *vp, *kq, *vq;
    if constexpr (UNI) {                                    // one page holds the unit
      const int at = __builtin_amdgcn_readfirstlane(4 * u), off = off_of(at);
      const int page = __builtin_amdgcn_readfirstlane(page_of(at));
      kp = cache.key(page, kvh, off, D) + (16 * (c >> 2) + (c & 3)) * D + 16 * g;
      vp = cache.values(page, kvh, off, D) + 16 * g * D + 16 * c;
      kq = cache.kscale(page, kvh, off) + 16 * (c >> 2);
      vq = cache.vscale(page, kvh, off) + 16 * g;
    } else {
      const int gk = min(4 * u + (c >> 2), last), gv = min(4 * u + g, last);
      const int pk = page_of(gk), pv = page_of(gv), ok = off_of(gk), ov = off_of(gv);
      kp = cache.key(pk, kvh, ok, D) + (c & 3) * D + 16 * g;
      vp = cache.values(pv, kvh, ov, D) + 16 * c;
      kq = cache.kscale(pk, kvh, ok);
      vq = cache.vscale(pv, kvh, ov);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < KC; ++i) x.k[j][i] = *reinterpret_cast<const uint4*>(kp + 4 * j * D + 64 * i);
    x.ks = *reinterpret_cast<const uint4*>(kq);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) x.v[dt] = *reinterpret_cast<const uint4*>(vp + 256 * dt);
    x.vs = *reinterpret_cast<const uint4*>(vq);
  };
  auto compute = [&](Unit& x, int u) {
    // scales of this lane's four key rows
    unsigned kb[4], worst = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      kb[j] = ((&x.ks.x)[j] >> (8 * (c & 3))) & 255u;
      worst = max(worst, kb[j]);
    }
    if (__any(worst == QUANT_POISON)) {                     // a token that is no number: every code of its key becomes one
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (kb[j] == QUANT_POISON) {
          kb[j] = 127;
#pragma unroll
          for (int i = 0; i < KC; ++i) x.k[j][i] = make_uint4(0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu);
        }
    }
    if (RU * (u + 1) > L) {                                 // keys past the end: whatever lies there, nothing of it is kept
      const int n = min(max(L - RU * u - 16 * g, 0), 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = min(max(n - 4 * j, 0), 4);
        const unsigned keep = k == 4 ? ~0u : (1u << (8 * k)) - 1;
        (&x.vs.x)[j] &= keep;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) (&x.v[dt].x)[j] &= keep;
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
        const bf16x8 a = quant_eight(x.k[j][i].x, x.k[j][i].y, ksc), b = quant_eight(x.k[j][i].z, x.k[j][i].w, ksc);
#pragma unroll
        for (int t = 0; t < NC; ++t) {
          sc[t][j] = mfma_bf16_k32(a, qf[t][2 * i], sc[t][j]);
          sc[t][j] = mfma_bf16_k32(b, qf[t][2 * i + 1], sc[t][j]);
        }
      }
    }
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
          p[t][j >> 1][4 * (j & 1) + i] = f2bf(e * quant_scale(((&x.vs.x)[j] >> (8 * i)) & 255u));
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
      const bf16x8 a = quant_eight(x.v[dt].x, x.v[dt].y, 1.f), b = quant_eight(x.v[dt].z, x.v[dt].w, 1.f);
#pragma unroll
      for (int t = 0; t < NC; ++t) {
        o[t][dt] = mfma_bf16_k32(a, p[t][0], o[t][dt]);
        o[t][dt] = mfma_bf16_k32(b, p[t][1], o[t][dt]);
      }
    }
  };
  Unit x;
  for (int u = ub + w; u < ue; u += RW) {
    load(x, u);
    compute(x, u);
  }

#pragma unroll
  for (int t = 0; t < NC; ++t) {
    const float lt = column_sum(l[t]);
    if (g == 0) sm[w][16 * t + c] = m[t], sl[w][16 * t + c] = lt;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) mfma_settle(o[t][dt]);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) so[w][16 * dt + 4 * g + i][16 * t + c] = o[t][dt][i];
  }
  __syncthreads();
  const long base = (((long)blockIdx.y * Hkv + kvh) * r.most + part) * (16 * NC);
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
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += so[k][d + i][col] * f;
    }
    if (parts > 1) {
      *reinterpret_cast<f32x4*>(r.po + (base + col) * D + d) = v;
      if (d == 0) r.ml[base + col] = make_float2(mx, sum);
    } else {
      const float inv = sum != 0.f ? 1.f / sum : 0.f;
      bf16x4 y;
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = f2bf(v[i] * inv);
      *reinterpret_cast<bf16x4*>(r.out + (long)(q0 + col / G) * r.out_stride + (long)(kvh * G + col % G) * D + d) = y;
    }
  }
}

template <int D, int NC>
__global__ void __launch_bounds__(256)
quant_rows_merge_kernel(Rows r, int Hkv) {
  const int kvh = blockIdx.x, G = r.Hq / Hkv;
  const int s = r.list ? r.list[blockIdx.y] : blockIdx.y;
  const int L = r.lens[s], q0 = r.cu ? r.cu[s] : s, qlen = r.cu ? r.cu[s + 1] - q0 : 1, nrow = min(qlen * G, 16 * NC);
  const int parts = rows_parts(r, rows_span(r, L, qlen).units, rows_per(r, Hkv));
  if (parts == 1) return;
  const long base = ((long)blockIdx.y * Hkv + kvh) * r.most * (16 * NC);
  for (int id = threadIdx.x; id < nrow * (D / 4); id += 256) {
    const int col = id / (D / 4), d = id % (D / 4) * 4;
    float m = -INFINITY, l = 0.f;
    f32x4 v{0.f, 0.f, 0.f, 0.f};
    for (int p0 = 0; p0 < parts; p0 += 4) {
      float2 x[4];
      f32x4 y[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {                         // (a part past the last: the last one, weight 0)
        const long at = base + (long)min(p0 + k, parts - 1) * (16 * NC) + col;
        x[k] = r.ml[at];
        y[k] = *reinterpret_cast<const f32x4*>(r.po + at * D + d);
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
        if (p0 + k >= parts) break;
        const float f = __builtin_amdgcn_exp2f(x[k].x - use);
        l += x[k].y * f;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += y[k][i] * f;
      }
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
    bf16x4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = f2bf(v[i] * inv);
    *reinterpret_cast<bf16x4*>(r.out + (long)(q0 + col / G) * r.out_stride + (long)(kvh * G + col % G) * D + d) = y;
  }
}

}  // namespace

// n sequences (list names them, or the first n), each with at most 16 * tiles rows (query, head of a kv head); most: parts a
// sequence at most, per: units of 64 keys a part (0: the kernel's own cut); ws: n * Hkv * most * 16 * tiles * (D + 2) floats.
EIA_API int eia_quant_rows(const void* q, long q_stride, void* out, long out_stride, const void* k, const void* v, const void* ks,
                           const void* vs, long codes, long scales, const int* tables, int bt_stride, const int* lens, const int* cu,
                           const int* list, int n, float scale, int Hq, int Hkv, int D, int bs, int causal, int window, int chunk,
                           int tiles, int most, int per, int slots, float* ws, hipStream_t st) {
  if (n < 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || bs <= 0 || bs % QUANT_GROUP || most < 1 || (most > 1 && !ws) || n > 65535 || most > 65535 ||
      slots < 1 || tiles < 1)
    return EIA_BAD_SHAPE;
  if (n == 0) return EIA_OK;
  const int groups = bs / QUANT_GROUP;
  const long sums = (long)n * Hkv * most * 16 * tiles * D;
  const Rows r{(const bf16_t*)q, (bf16_t*)out, q_stride, out_stride, tables, lens, cu, list, bt_stride, n, Hq, causal, window, chunk,
               scale * FLASH_LOG2E, ws, reinterpret_cast<float2*>(ws + sums), most, per, slots, groups,
               (unsigned)(((1ull << 32) + groups - 1) / groups)};
  const QuantCache c{(uint8_t*)k, (uint8_t*)v, (uint8_t*)ks, (uint8_t*)vs, codes, scales, Hkv, bs};
#define RW_GO(D, NC)                                                                                                       \
  do {                                                                                                                     \
    if (bs % RU == 0) hipLaunchKernelGGL((quant_rows_kernel<D, NC, true>), dim3(Hkv, n, most), dim3(64 * RW), 0, st, r, c); \
    else hipLaunchKernelGGL((quant_rows_kernel<D, NC, false>), dim3(Hkv, n, most), dim3(64 * RW), 0, st, r, c);             \
    if (most > 1) hipLaunchKernelGGL((quant_rows_merge_kernel<D, NC>), dim3(Hkv, n), dim3(256), 0, st, r, Hkv);             \
  } while (0)
  if (tiles > (D == 256 ? 1 : 2)) return EIA_UNSUPPORTED;   // (more do not fit the registers)
  switch (D) {
    case 64: if (tiles == 1) RW_GO(64, 1); else RW_GO(64, 2); break;
    case 128: if (tiles == 1) RW_GO(128, 1); else RW_GO(128, 2); break;
    case 256: RW_GO(256, 1); break;
    default: return EIA_UNSUPPORTED;
  }
#undef RW_GO
  EIA_LAUNCH_CHECK();
}
