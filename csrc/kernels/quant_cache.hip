// Writing and reading the 8-bit key/value cache (eia_quant.h).
//
// The write takes the QKV projection's rows [T, (Hq + 2 Hkv) D] (bf16, or the fp32 partial sums of a split-K GEMM):
// bias, RMS norm of queries and keys, rotation; queries go on in bf16, keys and values into the cache.  All of it
// rounded once: queries are formed in fp32, keys in fp64, values are the projection's own and a bias.
//
// A head of a token is D / 16 lanes, sixteen values a lane (two halves of eight, as they rotate); the lanes of a kv head
// hold the key row and the value row, because a value that is not finite marks both.  A workgroup takes TT tokens and
// 64 / (D / 16) query heads, or as many kv heads as fill it.  Codes of values go through LDS so that sixteen tokens of a
// channel are stored together where their slots are (a prompt's are, but for its first and last group).
//
// Both are bound by memory where they are large.  32 heads on 8 of 128: 4096 tokens written 20.8 us, 4.5 TB/s read and written (a copy
// of 2 GiB 4.87), 8192 40.0, 4.7; 32768 rows read back 40 us, 5.0 TB/s.  Few tokens are a launch and a chain of two loads: 32 written 4.4 us,
// 200 read 3.6.  Four heads a thread share a token's angles, which are as many bytes as two heads: 4096 tokens 21.8 -> 20.4.
#include "eia_quant.h"

namespace {

struct QuantSrc {
  const bf16_t* qkv;       // [T][stride], or
  const float* part;       // split-K sums [sk][T][(Hq + 2 Hkv) D]
  long stride, slab;
  int sk;
  const bf16_t *bias, *q_norm, *k_norm;
  float eps;
};

template <int D, bool NEOX> EIA_DEV void halves_of(int sub, int& e0, int& e1) {
  e0 = NEOX ? 8 * sub : 16 * sub;
  e1 = NEOX ? D / 2 + 8 * sub : 16 * sub + 8;
}

// Sixteen values of a head's row, with the bias: asked for, and taken.
template <int D, bool NEOX, bool ONCE> struct RowLoad {
  bf16x8 v[2], b[2];
  EIA_DEV void ask(const QuantSrc& src, int t, int head, int sub) {
    int e[2];
    halves_of<D, NEOX>(sub, e[0], e[1]);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (!src.part) v[h] = __builtin_bit_cast(bf16x8, quant_load<ONCE>(src.qkv + (long)t * src.stride + (long)head * D + e[h]));
      if (src.bias) b[h] = *reinterpret_cast<const bf16x8*>(src.bias + (long)head * D + e[h]);
    }
  }
  EIA_DEV void take(const QuantSrc& src, int t, int head, int ntot, int sub, float (&x)[16]) {
    int e[2];
    halves_of<D, NEOX>(sub, e[0], e[1]);
    if (src.part) {
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = 0.f;
      for (int k = 0; k < src.sk; ++k) {
        const float* p = src.part + k * src.slab + ((long)t * ntot + head) * D;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const f32x4 y = *reinterpret_cast<const f32x4*>(p + e[h] + 4 * q);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[8 * h + 4 * q + j] += y[j];
          }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = bf2f(v[j / 8][j % 8]);
    }
    if (src.bias) {
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] += bf2f(b[j / 8][j % 8]);
    }
  }
};

// T: queries are rounded to bf16 and formed in fp32; keys in fp64 (their codes are borders apart, and the heads are few), so that a code
// is the nearest to what bias, norm and rotation of the projection's numbers give.
template <int D, bool NEOX, typename T>
EIA_DEV void norm_row(const bf16_t* w, float eps, int sub, T (&x)[16]) {
  T ss = 0;
#pragma unroll
  for (int j = 0; j < 16; ++j) ss += x[j] * x[j];
#pragma unroll
  for (int o = 1; o < D / 16; o <<= 1) ss += __shfl_xor(ss, o, 64);
  const T inv = (T)1 / sqrt(ss / (T)D + (T)eps);
  int e[2];
  halves_of<D, NEOX>(sub, e[0], e[1]);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const bf16x8 v = *reinterpret_cast<const bf16x8*>(w + e[h]);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[8 * h + j] *= inv * (T)bf2f(v[j]);
  }
}

// A token's cos and sin for a lane's eight pairs: cs is cos [D / 2] | sin [D / 2].
template <int D> struct Turn {
  float c[8], s[8];
  EIA_DEV void ask(const float* cs, int sub) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(cs + 8 * sub + 4 * q), b = *reinterpret_cast<const f32x4*>(cs + D / 2 + 8 * sub + 4 * q);
#pragma unroll
      for (int j = 0; j < 4; ++j) c[4 * q + j] = a[j], s[4 * q + j] = b[j];
    }
  }
  template <bool NEOX, typename T> EIA_DEV void rotate(T (&x)[16]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      T &a = x[NEOX ? j : 2 * j], &b = x[NEOX ? 8 + j : 2 * j + 1];
      const T ra = fma(a, (T)c[j], -(b * (T)s[j])), rb = fma(b, (T)c[j], a * (T)s[j]);
      a = ra;
      b = rb;
    }
  }
};

template <int D, bool NEOX, int TT, int NH, bool ONCE>
__global__ void __launch_bounds__(256)
quant_write_kernel(QuantSrc src, const int* __restrict__ positions, const float* __restrict__ cos_sin, unsigned last_angle,
                   const int* __restrict__ slots, QuantCache cache, long num_slots, bf16_t* __restrict__ q_out, int T, int Hq,
                   int q_groups) {
  constexpr int TPH = D / 16, HPB = 256 / TPH / TT;        // lanes of a head, heads of a workgroup
  static_assert(HPB >= 1, "");
  const int sub = threadIdx.x % TPH, at = threadIdx.x / TPH;
  const int i = at % TT, Hkv = cache.Hkv, ntot = Hq + 2 * Hkv;
  int e0, e1;
  halves_of<D, NEOX>(sub, e0, e1);
  if ((int)blockIdx.y < q_groups) {
    const int t = blockIdx.x * TT + i;
    const int h0 = blockIdx.y * HPB * NH + at / TT;        // heads h0, h0 + HPB, ...: one token's angles for all of them
    if (t >= T || h0 >= Hq) return;                        // (a head's lanes together)
    RowLoad<D, NEOX, ONCE> row[NH];
    Turn<D> turn;
#pragma unroll
    for (int n = 0; n < NH; ++n) row[n].ask(src, t, min(h0 + n * HPB, Hq - 1), sub);
    if (cos_sin) turn.ask(cos_sin + (long)min((unsigned)positions[t], last_angle) * D, sub);
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      const int h = h0 + n * HPB;
      if (h >= Hq) break;
      float x[16];
      row[n].take(src, t, h, ntot, sub, x);
      if (src.q_norm) norm_row<D, NEOX>(src.q_norm, src.eps, sub, x);
      if (cos_sin) turn.template rotate<NEOX>(x);
      bf16x8 a, b;
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] = f2bf(x[j]), b[j] = f2bf(x[8 + j]);
      bf16_t* o = q_out + ((long)t * Hq + h) * D;
      *reinterpret_cast<bf16x8*>(o + e0) = a;
      *reinterpret_cast<bf16x8*>(o + e1) = b;
    }
    return;
  }
  __shared__ __align__(16) uint8_t tile[HPB][D][TT];
  // (Tiles that begin with the first slot's group, as the read's, wait for that slot before their rows: 4096 tokens from a group's
  // first slot on 20.2 -> 22.2 us, from its sixth 23.4 -> 22.5.)
  const int t0 = blockIdx.x * TT, t = t0 + i;
  const int hh = at / TT, h = (blockIdx.y - q_groups) * HPB + hh;
  const long slot = t < T ? slots[t] : -1;
  const bool live = slot >= 0 && slot < num_slots && h < Hkv;
  RowLoad<D, NEOX, ONCE> krow, vrow;
  Turn<D> turn;
  if (t < T && h < Hkv) {                                  // (whatever the slot: rows are asked for beside it)
    krow.ask(src, t, Hq + h, sub);
    vrow.ask(src, t, Hq + Hkv + h, sub);
    if (cos_sin) turn.ask(cos_sin + (long)min((unsigned)positions[t], last_angle) * D, sub);
  }
  if (live) {
    float k[16], v[16];
    krow.take(src, t, Hq + h, ntot, sub, k);
    vrow.take(src, t, Hq + Hkv + h, ntot, sub, v);
    if (src.k_norm || cos_sin) {
      double x[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = k[j];
      if (src.k_norm) norm_row<D, NEOX>(src.k_norm, src.eps, sub, x);
      if (cos_sin) turn.template rotate<NEOX>(x);
#pragma unroll
      for (int j = 0; j < 16; ++j) k[j] = quant_odd(x[j]);
    }
    // magnitudes as bits: what is not finite is the largest
    unsigned mk = 0, mv = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      mk = max(mk, __float_as_uint(k[j]) & 0x7fffffffu);
      mv = max(mv, __float_as_uint(v[j]) & 0x7fffffffu);
    }
#pragma unroll
    for (int o = 1; o < TPH; o <<= 1) {
      mk = max(mk, (unsigned)__shfl_xor((int)mk, o, 64));
      mv = max(mv, (unsigned)__shfl_xor((int)mv, o, 64));
    }
    const bool poison = max(mk, mv) >= 0x7f800000u;
    const unsigned bk = poison ? QUANT_POISON : quant_byte(mk), bv = poison ? 127 : quant_byte(mv);
    const int page = (int)(slot / cache.bs), off = (int)(slot % cache.bs);
    unsigned w[4], u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = poison ? 0 : quant_pack(k[4 * j], k[4 * j + 1], k[4 * j + 2], k[4 * j + 3], quant_inverse(bk));
      u[j] = poison ? 0 : quant_pack(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3], quant_inverse(bv));
    }
    uint8_t* kp = cache.key(page, h, off, D);
    *reinterpret_cast<uint2*>(kp + e0) = make_uint2(w[0], w[1]);
    *reinterpret_cast<uint2*>(kp + e1) = make_uint2(w[2], w[3]);
    if (sub == 0) {
      *cache.kscale(page, h, off) = (uint8_t)bk;
      *cache.vscale(page, h, off) = (uint8_t)bv;
    }
    if constexpr (TT == QUANT_GROUP) {
#pragma unroll
      for (int j = 0; j < 16; ++j) tile[hh][j < 8 ? e0 + j : e1 + j - 8][i] = (uint8_t)(u[j / 4] >> (8 * (j & 3)));
    } else {
      uint8_t* vp = cache.values(page, h, off & ~(QUANT_GROUP - 1), D) + off % QUANT_GROUP;
#pragma unroll
      for (int j = 0; j < 16; ++j) vp[QUANT_GROUP * (j < 8 ? e0 + j : e1 + j - 8)] = (uint8_t)(u[j / 4] >> (8 * (j & 3)));
    }
  }
  if constexpr (TT == QUANT_GROUP) {
    __syncthreads();
    // whole groups: their first slot is a multiple of 16 and the others follow (the same for the whole workgroup)
    const int lane = threadIdx.x & 15;
    const int mine = t0 + lane < T ? slots[t0 + lane] : -1, first = __builtin_amdgcn_readfirstlane(mine);
    const bool whole = __all(mine == first + lane) && first >= 0 && first % QUANT_GROUP == 0 && (long)first + QUANT_GROUP <= num_slots;
    if (whole) {
      const int page = first / cache.bs, off = first % cache.bs;
      for (int r = threadIdx.x; r < HPB * D; r += 256) {
        const int g = (blockIdx.y - q_groups) * HPB + r / D;
        if (g < Hkv) *reinterpret_cast<uint4*>(cache.values(page, g, off, D) + QUANT_GROUP * (r % D)) = *reinterpret_cast<const uint4*>(&tile[r / D][r % D][0]);
      }
    } else {
      const bool there = mine >= 0 && mine < num_slots;
      const int page = there ? mine / cache.bs : 0, off = there ? mine % cache.bs : 0;
      for (int r = threadIdx.x / 16; r < HPB * D; r += 16) {
        const int g = (blockIdx.y - q_groups) * HPB + r / D;
        if (g < Hkv && there) cache.values(page, g, off & ~(QUANT_GROUP - 1), D)[QUANT_GROUP * (r % D) + off % QUANT_GROUP] = tile[r / D][r % D][lane];
      }
    }
  }
}

// Rows of sixteen slots and one head a workgroup part: keys straight through, values through LDS as the cache holds them.
// Rows of slots outside the cache are zeros.  Tiles begin with the first slot's group, so that rows in order meet whole groups: 777
// from a group's third slot on 5.9 -> 3.8 us.
template <int D, bool ONCE>
__global__ void __launch_bounds__(256)
quant_read_kernel(QuantCache cache, const int* __restrict__ slots, long num_slots, int n, bf16_t* __restrict__ k_out, bf16_t* __restrict__ v_out) {
  constexpr int TPH = D / 16, HPB = 256 / TPH / QUANT_GROUP;
  __shared__ __align__(16) uint8_t tile[HPB][D * QUANT_GROUP];
  const int t0 = blockIdx.x * QUANT_GROUP - max(slots[0], 0) % QUANT_GROUP, Hkv = cache.Hkv, h0 = blockIdx.y * HPB;
  const int lane = threadIdx.x & 15;
  const bool asked = t0 + lane >= 0 && t0 + lane < n;
  const int mine = asked ? slots[t0 + lane] : -1;
  const bool there = mine >= 0 && mine < num_slots;
  // tokens of one group at their places in it (the tile's ends may hold others' slots)
  const unsigned long long some = __ballot(there);
  const int base = __shfl(mine - lane, some ? __builtin_ctzll(some) : 0, 64);
  const bool whole = some && __all(!there || mine - lane == base) && base >= 0 && base % QUANT_GROUP == 0;
  constexpr int N = HPB * D / QUANT_GROUP;
  if (whole) {
    const int page = base / cache.bs, off = base % cache.bs;
#pragma unroll
    for (int r = threadIdx.x; r < HPB * D; r += 256)
      if (h0 + r / D < Hkv)
        *reinterpret_cast<uint4*>(&tile[r / D][QUANT_GROUP * (r % D)]) = quant_load<ONCE>(cache.values(page, h0 + r / D, off, D) + QUANT_GROUP * (r % D));
  } else {
    const int page = there ? mine / cache.bs : 0, off = there ? mine % cache.bs : 0;
    uint8_t x[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int r = threadIdx.x / QUANT_GROUP + 16 * k;
      x[k] = there && h0 + r / D < Hkv ? cache.values(page, h0 + r / D, off & ~(QUANT_GROUP - 1), D)[QUANT_GROUP * (r % D) + off % QUANT_GROUP] : 0;
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int r = threadIdx.x / QUANT_GROUP + 16 * k;
      tile[r / D][QUANT_GROUP * (r % D) + lane] = x[k];
    }
  }
  __syncthreads();
  const int sub = threadIdx.x % TPH, i = threadIdx.x / TPH % QUANT_GROUP, hh = threadIdx.x / TPH / QUANT_GROUP, h = h0 + hh, t = t0 + i;
  if (t < 0 || t >= n || h >= Hkv) return;
  const long slot = slots[t];
  const bool live = slot >= 0 && slot < num_slots;
  const int page = live ? (int)(slot / cache.bs) : 0, off = live ? (int)(slot % cache.bs) : 0;
  const unsigned bk = live ? *cache.kscale(page, h, off) : 127, bv = live ? *cache.vscale(page, h, off) : 127;
  uint4 w = live ? quant_load<ONCE>(cache.key(page, h, off, D) + 16 * sub) : make_uint4(0, 0, 0, 0), u;
  unsigned x[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[j] = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) x[j] |= (unsigned)tile[hh][QUANT_GROUP * (16 * sub + 4 * j + b) + i] << (8 * b);
  }
  u = live ? make_uint4(x[0], x[1], x[2], x[3]) : make_uint4(0, 0, 0, 0);
  if (bk == QUANT_POISON) w = u = make_uint4(0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu);
  const float sk = bk == QUANT_POISON ? 1.f : quant_scale(bk), sv = quant_scale(bv);
  const long o = ((long)t * Hkv + h) * D + 16 * sub;
  *reinterpret_cast<bf16x8*>(k_out + o) = quant_eight(w.x, w.y, sk);
  *reinterpret_cast<bf16x8*>(k_out + o + 8) = quant_eight(w.z, w.w, sk);
  *reinterpret_cast<bf16x8*>(v_out + o) = quant_eight(u.x, u.y, sv);
  *reinterpret_cast<bf16x8*>(v_out + o + 8) = quant_eight(u.z, u.w, sv);
}

}  // namespace

// qkv bf16 rows, or part != nullptr: fp32 sums [sk][T][(Hq + 2 Hkv) D].  cos_sin [angles][D], nullptr: no rotation; positions are held
// to its rows.
EIA_API int eia_quant_write(const void* qkv, long qkv_stride, const float* part, int sk, const int* positions, const float* cos_sin,
                            int angles, const int* slots, void* k, void* v, void* ks, void* vs, long codes, long scales, int pages, void* q_out,
                            const void* bias, const void* q_norm, const void* k_norm, float eps, int T, int Hq, int Hkv, int D, int bs,
                            int neox, hipStream_t st) {
  if (T < 0 || Hq <= 0 || Hkv <= 0 || bs <= 0 || bs % QUANT_GROUP || (part && sk < 1) || (!q_norm) != (!k_norm) ||
      (cos_sin && angles < 1))
    return EIA_BAD_SHAPE;
  if (T == 0) return EIA_OK;
  const QuantSrc src{(const bf16_t*)qkv, part, qkv_stride, (long)T * (Hq + 2 * Hkv) * D, sk, (const bf16_t*)bias, (const bf16_t*)q_norm,
                     (const bf16_t*)k_norm, eps};
  const QuantCache c{(uint8_t*)k, (uint8_t*)v, (uint8_t*)ks, (uint8_t*)vs, codes, scales, Hkv, bs};
#define QW_GO(D, NX, TT, NH, ONCE)                                                                                                      \
  do {                                                                                                                            \
    constexpr int hpb = 256 / (D / 16) / TT;                                                                                      \
    const int qg = (Hq + hpb * NH - 1) / (hpb * NH);                                                                              \
    hipLaunchKernelGGL((quant_write_kernel<D, NX, TT, NH, ONCE>), dim3((T + TT - 1) / TT, qg + (Hkv + hpb - 1) / hpb), dim3(256), 0, st, src, \
                       positions, cos_sin, angles - 1u, slots, c, (long)pages * bs, (bf16_t*)q_out, T, Hq, qg);                                \
  } while (0)
#define QW_N(D, NX)                                    \
  do {                                                 \
    if (T < 256) QW_GO(D, NX, 1, 1, false);            \
    else if (once) QW_GO(D, NX, 16, 4, true);          \
    else QW_GO(D, NX, 16, 4, false);                   \
  } while (0)
#define QW_D(D) do { if (neox) QW_N(D, true); else QW_N(D, false); } while (0)
  // Rows of more than a quarter of the last cache (256 MB) are read past the caches.  32 heads on 8 of 128, us as usual / past them: 4096
  // tokens (48 MiB) 20.4 / 21.0, 8192 46.1 / 39.3, 32768 184 / 172; 12 on 4 of 256, 8192 (80 MiB) 37.7 / 33.2; 12 of 64, 8192 (36 MiB) 15.8 /
  // 19.0.
  // Fewer than 256 tokens go a token a workgroup row, each with a head a thread; from there on sixteen tokens share a tile, which a whole group
  // stores in 16-byte pieces and a group in part, in 1.3 us more, by bytes.  us, 32 heads on 8 of 128, a token a row / sixteen from a group's
  // first slot on / from its sixth: 64 tokens 4.2 / 4.2 / 5.7, 128 4.5 / 4.3 / 5.8, 192 4.9 / 4.4 / 5.9, 255 5.2 / 5.7 / 6.0, 256 5.2 / 4.5 / 6.0, 384 6.6 /
  // 4.7 / 6.3, 512 7.4 / 5.1 / 6.7; 12 of 64: 192 4.4 / 4.0 / 5.4, 384 5.5 / 4.0 / 5.5; 12 on 4 of 256: 192 5.1 / 4.8 / 5.8, 384 6.8 / 5.0 / 6.2.
  // Heads a thread, one / two / four: 32 on 8 of 128, 512 tokens 5.5 / 5.2 / 5.1, 1024 9.1 / 7.3 / 7.3, 2048 13.9 / 13.0 / 11.0; 28 on 4 with bias and
  // norms, 777 7.8 / 7.6 / 7.9, 2048 11.1 / 11.5 / 10.8; 12 on 4 of 256, 777 7.6 / 7.4 / 7.4.
  const bool once = (long)T * (Hq + 2 * Hkv) * D * 2 > 64l << 20;
  switch (D) {
    case 64: QW_D(64); break;
    case 128: QW_D(128); break;
    case 256: QW_D(256); break;
    default: return EIA_UNSUPPORTED;
  }
#undef QW_D
#undef QW_N
#undef QW_GO
  EIA_LAUNCH_CHECK();
}

EIA_API int eia_quant_read(const void* k, const void* v, const void* ks, const void* vs, long codes, long scales, int pages,
                           const int* slots, int n, void* k_out, void* v_out, int Hkv, int D, int bs, hipStream_t st) {
  if (n < 0 || Hkv <= 0 || bs <= 0 || bs % QUANT_GROUP) return EIA_BAD_SHAPE;
  if (n == 0) return EIA_OK;
  const QuantCache c{(uint8_t*)k, (uint8_t*)v, (uint8_t*)ks, (uint8_t*)vs, codes, scales, Hkv, bs};
  // As the write's: us as usual / past the caches, 8 heads of 128: 4096 rows (8 MiB) 8.5 / 8.7, 8192 11.9 / 13.7, 32768 (64 MiB) 46.9 / 39.9.
  const bool once = (long)n * Hkv * D * 2 > 32l << 20;
#define QR_GO(D)                                                                                                                   \
  do {                                                                                                                             \
    constexpr int hpb = 256 / (D / 16) / QUANT_GROUP;                                                                              \
    auto* f = once ? quant_read_kernel<D, true> : quant_read_kernel<D, false>;                                                     \
    hipLaunchKernelGGL(f, dim3((n + 2 * QUANT_GROUP - 2) / QUANT_GROUP, (Hkv + hpb - 1) / hpb), dim3(256), 0, st, c, slots,            \
                       (long)pages * bs, n, (bf16_t*)k_out, (bf16_t*)v_out);                                                       \
  } while (0)
  switch (D) {
    case 64: QR_GO(64); break;
    case 128: QR_GO(128); break;
    case 256: QR_GO(256); break;
    default: return EIA_UNSUPPORTED;
  }
#undef QR_GO
  EIA_LAUNCH_CHECK();
}
