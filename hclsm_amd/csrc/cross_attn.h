// Shared pieces of the cross-attention kernels: arguments, operand traits, LDS tiles.
//
// One unit of work is a batch row and one key head.  The G = H / Hk query heads that read a key head are rows of one
// product: row r of a unit is query r / G of head hk G + r % G, so shared heads cost no further pass over the keys
// and their gradients are sums over rows like any other.
//
// Every product is formed transposed so that a lane owns one query row or one key (li = lane % 16) in all of them
// (g = lane / 16):
//   S^T = K Q^T     16 x 16 tile: the lane holds keys 4g .. 4g + 3 of its row li,
//   O^T = V^T P^T   those values, rounded, are the second operand as they stand: the contraction runs over the keys in
//                   the order 4g + r of one tile (float32) or of a pair of tiles (16 bits), and V^T is read in that
//                   order (ds_read_b64_tr_b16: lane li gets rows 4g .. 4g + 3 of column li),
// and the same with rows and keys exchanged for the gradients of k and v.
#pragma once

#include "internal.h"

namespace hclsm {

typedef float caf4 __attribute__((ext_vector_type(4)));
typedef __bf16 cab8 __attribute__((ext_vector_type(8)));
typedef _Float16 cah8 __attribute__((ext_vector_type(8)));
typedef short cas4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) cas4 ca_lds_s4;
typedef __attribute__((address_space(3))) void ca_lds_void;

struct CaArgs {
  const char *q, *k, *v, *g;        // inputs; gradient of the output
  char *o, *olo, *dq, *dk, *dv;     // contiguous [B, Lq, H, dh] / [B, Lk, Hk, dh]
  float* lse;                       // [B, H, Lq] natural logarithm, -inf for rows without keys
  float* delta;                     // [B, H, Lq] sum(g o), written by the dq kernel for the dk, dv kernel
  float* part;                      // partial sums of a split launch
  float* part_lse;                  // forward: log2 of the partial denominators
  int64_t qsb, qsl, qsh, ksb, ksl, ksh, vsb, vsl, vsh, gsb, gsl, gsh;   // element strides
  const uint8_t* pad;               // [B, Lk] nonzero: key not read; nullable
  int64_t psb;
  const void *klens, *qlens;        // [B] live keys / queries, nullable
  int klens64, qlens64;
  int Hk, G, Lq, Lk, dh;
  uint32_t gmul;                    // row / G = (row * gmul) >> 32 >> gshift (G > 1)
  int gshift;
  int units, tiles, nsplit, by_xcd;
  float scale, scale_log2;
};

// 16-byte operand fragments.  EPC: elements per 16 bytes; KS: contraction per fragment; NPT: 16-row tiles whose
// values make one fragment of a product over rows.
template <int DT> struct CaT;
template <> struct CaT<HCLSM_BF16> {
  using T = uint16_t;
  using Frag = cab8;
  static constexpr int EPC = 8, KS = 32, NPT = 2;
  static __device__ __forceinline__ caf4 mma(Frag a, Frag b, caf4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack2(float a, float b) { return pack_bf16x2(a, b); }
  static __device__ __forceinline__ float lo(uint32_t w) { return __uint_as_float(w << 16); }
  static __device__ __forceinline__ float hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
};
template <> struct CaT<HCLSM_F16> {
  using T = uint16_t;
  using Frag = cah8;
  static constexpr int EPC = 8, KS = 32, NPT = 2;
  static __device__ __forceinline__ caf4 mma(Frag a, Frag b, caf4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack2(float a, float b) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    h2 r;
    r.x = (_Float16)a;
    r.y = (_Float16)b;
    return __builtin_bit_cast(uint32_t, r);
  }
  static __device__ __forceinline__ float lo(uint32_t w) { return (float)__builtin_bit_cast(_Float16, (uint16_t)w); }
  static __device__ __forceinline__ float hi(uint32_t w) { return (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16)); }
};
template <> struct CaT<HCLSM_F32> {
  using T = float;
  using Frag = caf4;
  static constexpr int EPC = 4, KS = 16, NPT = 1;
  // element e of both operands is the contraction index 4g + e: any order will do as long as both use it
  static __device__ __forceinline__ caf4 mma(Frag a, Frag b, caf4 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};

template <int DT> __device__ __forceinline__ typename CaT<DT>::Frag ca_frag(uint4 w) {
  return __builtin_bit_cast(typename CaT<DT>::Frag, w);
}

// Fragment of the values of NPT tiles (t[0] alone for float32), rounded to the operand type.
template <int DT> __device__ __forceinline__ typename CaT<DT>::Frag ca_pack(const caf4* t) {
  if constexpr (DT == HCLSM_F32) {
    return t[0];
  } else {
    using A = CaT<DT>;
    const uint4 w = {A::pack2(t[0][0], t[0][1]), A::pack2(t[0][2], t[0][3]), A::pack2(t[1][0], t[1][1]),
                     A::pack2(t[1][2], t[1][3])};
    return ca_frag<DT>(w);
  }
}

// The same in PARTS operands: the rounded values, and with 2 what the rounding dropped (zero where they overflow).
// A product over both has the values to 2^-16 (bf16) or 2^-22 (fp16, or its smallest step).
template <int DT, int PARTS> __device__ __forceinline__ void ca_pack_parts(const caf4* t, typename CaT<DT>::Frag* out) {
  out[0] = ca_pack<DT>(t);
  if constexpr (PARTS == 2) {
    using A = CaT<DT>;
    const uint4 w = __builtin_bit_cast(uint4, out[0]);
    const uint32_t h[4] = {w.x, w.y, w.z, w.w};
    caf4 rest[2];
#pragma unroll
    for (int i = 0; i < 8; ++i) {       // (infinities have no rest)
      const float d = t[i >> 2][i & 3] - (i & 1 ? A::hi(h[i >> 1]) : A::lo(h[i >> 1]));
      rest[i >> 2][i & 3] = fabsf(d) < INFINITY ? d : 0.f;
    }
    out[1] = ca_pack<DT>(rest);
  }
}

// A row's exponentials are taken against a reference (log2): its lowest value, which no score reaches from below; how far the
// row's maximum may pass it before it moves; and how far below the maximum it is put then.  float16 weights use the range
// up to 2^15: what lies 2^36 below the largest weight is lost (with the largest at one it would be what lies 2^25 below, and
// where one key of a hundred thousand stands out that adds up to 2^-8 of the softmax).
constexpr float CA_LOW = -3.0e38f;
template <int DT> constexpr float CA_SLACK = DT == HCLSM_F16 ? 15.f : 8.f;
template <int DT> constexpr float CA_BELOW = DT == HCLSM_F16 ? 11.f : 0.f;

// Maxima that pass a NaN on (v_maximum3_f32: one instruction for two values, and no step to quiet its operands first).
__device__ __forceinline__ float ca_max3(float a, float b, float c) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}
// over the four lanes that share a row, as rows4_max
__device__ __forceinline__ float ca_rows4_max(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __builtin_elementwise_maximum(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __builtin_elementwise_maximum(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Scores' gradients ds = p (dP - delta) of a row lie around |g| / Lk, which float16 (2^-24 to 65504) does not hold for small g
// or many keys, nor for large g and v.  They are rounded as ds times a power of two, one for each row of dq and each key
// of dk (a lane's own result column, so the factor leaves the sum again exactly): it starts at 2^CA_F16_START and is lowered,
// the sums so far with it, when a value would pass 2^15, so that the largest one lies at 2^10 or above and values down to
// 2^-24 of it keep all their bits.  The rms error of dq and dk is then 1.41 times that of the results' rounding for g of any size (two
// operands: 1.0), where plain rounding gave 5 to 22 times for g of 1e-3 and 4096 to 32768 keys.  Measured (us, without and
// with it): 8 x 1024 queries, 2048 keys, 12 heads of 64: dq 93, 104, dk and dv 118, 128; of 128 on 4: 205, 220 and 269, 293;
// 256 frames, 32 slots, 196 tokens, 6 heads of 64: 50, 52.
template <int DT> constexpr bool CA_RANGED = DT == HCLSM_F16;
constexpr float CA_F16_MOST = 32768.f;
constexpr int CA_F16_EXP = 11, CA_F16_START = 32;      // values are brought below 2^11
__device__ __forceinline__ float ca_pow2(int e) { return __builtin_ldexpf(1.f, e); }
// Weights p are rounded for the gradient of v as p 2^12 (the log-sum lowered by as much), so that they keep all their bits
// down to 2^-26, the even weight of 67 million keys; p itself would have lost some from 16 thousand keys on.  A p past one,
// from scores so large that float32 does not hold their differences, may be 2^4 before it overflows.
template <int DT> constexpr float CA_P_SHIFT = DT == HCLSM_F16 ? 12.f : 0.f;
template <int DT> constexpr float CA_P_DOWN = DT == HCLSM_F16 ? 0x1p-12f : 1.f;
// N tiles of a row's values times up; the largest magnitude among them (NaN where there is one).
template <int N> __device__ __forceinline__ float ca_scale_most(caf4* v, float up) {
  float m = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    v[k] *= up;
#pragma unroll
    for (int r = 0; r < 4; r += 2) m = ca_max3(m, fabsf(v[k][r]), fabsf(v[k][r + 1]));
  }
  return m;
}
// The power of two that brings m to 2^10 .. 2^11 where it is past 2^15; 1 elsewhere, and for infinities and NaN.
__device__ __forceinline__ float ca_lowered(float m) {
  return m > CA_F16_MOST && m < INFINITY ? ca_pow2(CA_F16_EXP - __builtin_amdgcn_frexp_expf(m)) : 1.f;
}
// The same for any m, up to a factor of 2^64.
__device__ __forceinline__ float ca_fitted(float m) {
  const int e = CA_F16_EXP - __builtin_amdgcn_frexp_expf(m);
  return m > 0.f && m < INFINITY ? ca_pow2(e < 64 ? e : 64) : 1.f;
}
// 1 / f of a power of two
__device__ __forceinline__ float ca_unscaled(float f) { return ca_pow2(1 - __builtin_amdgcn_frexp_expf(f)); }

// sum over the elements of a 16-byte chunk of a * b
template <int DT> __device__ __forceinline__ float ca_dot(uint4 a, uint4 b, float s) {
  const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == HCLSM_F32) {
      s += __uint_as_float(x[i]) * __uint_as_float(y[i]);
    } else {
      s += CaT<DT>::lo(x[i]) * CaT<DT>::lo(y[i]);
      s += CaT<DT>::hi(x[i]) * CaT<DT>::hi(y[i]);
    }
  }
  return s;
}

// Four consecutive elements of an output row.
template <int DT> __device__ __forceinline__ void ca_store4(char* base, int64_t i, caf4 v) {
  if constexpr (DT == HCLSM_F32) {
    *reinterpret_cast<caf4*>(base + i * 4) = v;
  } else {
    const uint2 w = {CaT<DT>::pack2(v[0], v[1]), CaT<DT>::pack2(v[2], v[3])};
    *reinterpret_cast<uint2*>(base + i * 2) = w;
  }
}

// Rows of DH elements in LDS, as 16-byte chunks.  Two reads have to be free of bank conflicts: 16 rows at one chunk
// (operands along a row), and 32 bytes of each of 8 rows (the transposing read).  Rows of 8, 16 or 32 chunks of 16-bit
// elements exchange their chunks by the row's low three bits (measured: no conflict cycles); others are padded by one chunk.
template <int DT, int DH> struct CaTile {
  static constexpr int CH = DH / CaT<DT>::EPC;
  static constexpr bool XOR = DT != HCLSM_F32 && (CH == 8 || CH == 16 || CH == 32);
  static constexpr int PC = XOR ? CH : CH + 1;      // chunks of a row in LDS
  static constexpr int STRIDE = PC * 16;
  static __device__ __forceinline__ int swap(int row) { return !XOR ? 0 : CH == 8 ? row & 7 : (row & 7) << 1; }
  static __device__ __forceinline__ int off(int row, int chunk) { return row * STRIDE + ((chunk ^ swap(row)) << 4); }
  // bytes of a tile of `rows`, in whole transfers of a workgroup of `threads`
  static constexpr int bytes(int rows, int threads) { return (rows * PC + threads - 1) / threads * threads * 16; }
  // operand with rows row0 + li as its free index and elements KS c + 4 or 8 g .. of the row as contraction
  static __device__ __forceinline__ typename CaT<DT>::Frag frag(const char* t, int row0, int c, int li, int g) {
    return ca_frag<DT>(*reinterpret_cast<const uint4*>(t + off(row0 + li, 4 * c + g)));
  }
  // operand with columns 16 dt + li as its free index and rows row0 + 4g .. + 3 (and row0 + 16 + 4g ..) as contraction
  static __device__ __forceinline__ typename CaT<DT>::Frag frag_t(char* t, int row0, int dt, int li, int g) {
    if constexpr (DT == HCLSM_F32) {
      caf4 r;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        r[e] = *reinterpret_cast<const float*>(t + (row0 + 4 * g + e) * STRIDE + (16 * dt + li) * 4);
      return r;
    } else {
      const int row = row0 + 4 * g + (li >> 2), chunk = 2 * dt + ((li >> 1) & 1), sub = (li & 1) * 8;
      const cas4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ca_lds_s4*)(t + off(row, chunk) + sub));
      const cas4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ca_lds_s4*)(t + off(row + 16, chunk) + sub));
      typedef short s8 __attribute__((ext_vector_type(8)));
      const s8 r = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
      return __builtin_bit_cast(typename CaT<DT>::Frag, r);
    }
  }
};

// Four consecutive elements of the output, and what their rounding dropped where that is wanted.
template <int DT> __device__ __forceinline__ void ca_store_out(const CaArgs& a, int64_t i, caf4 v) {
  ca_store4<DT>(a.o, i, v);
  if constexpr (DT != HCLSM_F32) {
    if (a.olo != nullptr) {
      const uint32_t w0 = CaT<DT>::pack2(v[0], v[1]), w1 = CaT<DT>::pack2(v[2], v[3]);
      ca_store4<DT>(a.olo, i, caf4{v[0] - CaT<DT>::lo(w0), v[1] - CaT<DT>::hi(w0), v[2] - CaT<DT>::lo(w1), v[3] - CaT<DT>::hi(w1)});
    }
  }
}

__device__ __forceinline__ int ca_len(const void* lens, int is64, int64_t b, int most) {
  if (lens == nullptr) return most;
  const int64_t n = is64 ? reinterpret_cast<const int64_t*>(lens)[b] : (int64_t)reinterpret_cast<const int32_t*>(lens)[b];
  return n < 0 ? 0 : n > most ? most : (int)n;
}

// Unit, tile and split of a workgroup.  by_xcd: workgroup i runs on XCD i % 8, each with its own L2, so the
// tiles of one unit are given to one XCD and its keys (or rows) are fetched from HBM once.
struct CaWork {
  int unit, tile, split;
  int64_t b;
  int hk, rows, keys;       // live rows and keys (before the padding mask) of the unit
};

__device__ __forceinline__ bool ca_work(const CaArgs& a, CaWork& w) {
  const uint32_t per = (uint32_t)a.tiles * (uint32_t)a.nsplit;
  uint32_t i = blockIdx.x, rest;
  if (a.by_xcd) {
    const uint32_t j = i >> 3;
    w.unit = (int)((j / per) * 8 + (i & 7));
    rest = j % per;
  } else {
    w.unit = (int)(i / per);
    rest = i % per;
  }
  if (w.unit >= a.units) return false;
  w.split = (int)(rest / (uint32_t)a.tiles);
  w.tile = (int)(rest % (uint32_t)a.tiles);
  w.b = w.unit / a.Hk;
  w.hk = w.unit - (int)w.b * a.Hk;
  w.rows = ca_len(a.qlens, a.qlens64, w.b, a.Lq) * a.G;
  w.keys = ca_len(a.klens, a.klens64, w.b, a.Lk);
  return true;
}

__device__ __forceinline__ void ca_row(const CaArgs& a, int row, int& qi, int& hg) {
  qi = row;
  hg = 0;
  if (a.G > 1) {
    qi = (int)(__umulhi((uint32_t)row, a.gmul) >> a.gshift);
    hg = row - qi * a.G;
  }
}

// Rows of a tile of RR: whole queries where a query has no more heads than that.
__device__ __forceinline__ int ca_row_step(int G, int RR) { return G <= RR ? RR - RR % G : RR; }

// [begin, end) of a split's share of n, in whole multiples of `step` but for the end.
__device__ __forceinline__ void ca_range(int n, int nsplit, int split, int step, int& begin, int& end) {
  if (nsplit == 1) {
    begin = 0;
    end = n;
    return;
  }
  const int64_t share = ((int64_t)((n + step - 1) / step) + nsplit - 1) / nsplit * step;
  const int64_t b = share * split, e = b + share;
  begin = b < n ? (int)b : n;
  end = e < n ? (int)e : n;
}

// How a call is launched, a function of the sizes alone (the workspace is sized by the same rules).
struct CaPlan {
  int few;        // 0: tiles of many rows; 1, 2: at most 16 or 32 rows of a unit, ca_few_kernel (backward: ca_few_bwd_kernel)
  int nsplit;     // workgroups that share a unit's keys (out, dq); their results are joined by ca_join / ca_sum
  int nrows;      // backward: workgroups that share a unit's rows (dk, dv)
};
constexpr int CA_MAX_SPLIT = 256;
// Rows (in bytes, padded head) up to which ca_few_kernel is built for 16 rows and for 32 rows (float32, 16 bits), and
// ca_few_bwd_kernel: a step's keys and values, the accumulators and the queries all live in registers, and longer heads
// would spill.  Measured against the tiled kernels (us, 64 batch rows, 6 heads, 1500 keys; then 256 and 196): 1 row, bf16
// heads of 64: 29 against 28 and 17 against 19, of 128: 57, 54 and 32, 34, float32 of 64: 57, 110 and 31, 65; 32 rows:
// float32 of 64: 83, 109 and 52, 71, bf16 of 64: 44, 41 and 25, 24, where the weights keep their second operand for the
// difference, but of 128: 82, 68 and 70, 49, which take the tiles.  Backward of 32 rows: bf16 of 64: 95, 101 and 54, 67, of
// 128: 194, 236 and 125, 157; float32 of 64: 227, 406 and 121, 252.  Single float32 queries with heads past 128 take the
// tiles too: 64 x 1568 keys, 12 heads of 192: 570 us, of 256: 770, 3.2 TB/s, where heads of 128 take 211, 5.9 TB/s.
constexpr int CA_FEW1_BYTES = 512, CA_FEW2_F32_BYTES = 256, CA_FEW2_16BIT_BYTES = 128, CA_FEW_BWD_BYTES = 256;
constexpr int64_t ca_few2_bytes(int dtype) { return dtype == HCLSM_F32 ? CA_FEW2_F32_BYTES : CA_FEW2_16BIT_BYTES; }
constexpr int64_t ca_padded_dh(int64_t dh) {
  return dh <= 32 ? 32 : dh <= 64 ? 64 : dh <= 96 ? 96 : dh <= 128 ? 128 : dh <= 192 ? 192 : 256;
}
// Rows (or keys) of a workgroup's tile: 128, or 64 where there are no more or the operands are too wide for two 16-row
// tiles per wave.
constexpr int64_t ca_tile_rows(int64_t n, int64_t bytes) { return bytes <= 256 && n > 64 ? 128 : 64; }
// Weights and scores' gradients of 16-bit types are carried in two operands (the rounded values and what the rounding
// dropped) in the kernels for few rows, and in the tiled ones up to this many keys: there the roundings do not average
// out, and delta, which is a sum over the output and so over the forward's rounded weights, is as large as the terms it is
// taken from.  Errors of dq and dk against float64 went from up to 2.9 times to at most 1.5 times those of the results'
// own rounding (6700 and 2000 random calls).  It costs next to nothing there (us, bf16, one and two operands): 256 frames,
// 32 slots, 196 tokens, 6 heads of 64: backward 50.5, 53; 8 slots, heads of 128: 121, 126; 64 single queries on 1568 keys,
// 12 heads of 64: 50.8, 50.5; in tiles of 32 keys, 16 x 1024 queries, 32 keys, 12 heads of 64: 23.5 + 49.5, 22.3 + 49.8, of
// 128: 42.5 + 99.6, 40.6 + 85.4; of 256 with 512 queries: 43.0 + 95.1, 43.6 + 100.8.  For many rows and keys, where the
// products bound the kernels, results of either 16-bit type are off by 1.41 times their own rounding, and two operands
// would cost (forward, backward): 8 x 1024 queries, 2048 keys, 12 heads of 64: 65, 190 against 105, 280; of 128 on 4: 105,
// 389 against 178, 573; 8 x 2048 queries, 4099 keys: 180 against 282.
constexpr int CA_FINE_KEYS = 32;
CaPlan ca_forward_plan(int64_t B, int64_t Lq, int64_t Lk, int64_t Hk, int64_t G, int64_t dh, int dtype);
CaPlan ca_backward_plan(int64_t B, int64_t Lq, int64_t Lk, int64_t Hk, int64_t G, int64_t dh, int dtype);
int64_t ca_backward_bytes(const CaPlan& p, int64_t B, int64_t Lq, int64_t Lk, int64_t Hk, int64_t G, int64_t dh);
// out = partial outputs joined by their log-sums; sums of partial dq (keys = 0) or of dk and dv (keys = 1)
int ca_join(const CaArgs& a, int dtype, hipStream_t st);
int ca_sum(const CaArgs& a, int keys, int dtype, hipStream_t st);

// Host side: one launch per (element type, padded head size) is picked in cross_attn.hip.
int ca_forward_f32(CaArgs a, int64_t batch, void* ws, int64_t ws_bytes, hipStream_t st);
int ca_forward_bf16(CaArgs a, int64_t batch, void* ws, int64_t ws_bytes, hipStream_t st);
int ca_forward_f16(CaArgs a, int64_t batch, void* ws, int64_t ws_bytes, hipStream_t st);
int ca_backward_f32(CaArgs a, int64_t batch, void* ws, int64_t ws_bytes, hipStream_t st);
int ca_backward_bf16(CaArgs a, int64_t batch, void* ws, int64_t ws_bytes, hipStream_t st);
int ca_backward_f16(CaArgs a, int64_t batch, void* ws, int64_t ws_bytes, hipStream_t st);

}  // namespace hclsm
