// The chunked kernel of linear attention, instantiated for one element type per source file (linear_attn_*.hip).
#pragma once

#include "linear_attn.h"

namespace hclsm {

// Every matrix operand is a sum of bf16 planes, each the rounded rest of the ones before: a bf16 input is one, a float16
// input two (its 11 bits exactly), a float32 input three (24 bits).  What is computed in float32 in between (weights of
// pairs, the state) becomes two planes (2^-17 of the value; with one, results would be off by 1.4 times their own
// rounding) and three for float32; the state's own update has three planes of the weighted X, so that states are float32
// results.  bf16 has float32's range, so no value of any type needs a scale.
template <int DT> struct LaT;
template <> struct LaT<HCLSM_BF16> { static constexpr int NP = 1, NC = 2, RAW = 1; };
template <> struct LaT<HCLSM_F16> { static constexpr int NP = 2, NC = 2, RAW = 1; };
template <> struct LaT<HCLSM_F32> { static constexpr int NP = 3, NC = 3, RAW = 2; };

using LaB = CaT<HCLSM_BF16>;
using LaFrag = cab8;

// N planes of eight float32 values.
template <int N> __device__ __forceinline__ void la_split(const float* v, uint4* out) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = v[i];
#pragma unroll
  for (int p = 0; p < N; ++p) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = pack_bf16x2(r[2 * i], r[2 * i + 1]);
      if (p + 1 < N) {
        r[2 * i] -= LaB::lo(w[i]);
        r[2 * i + 1] -= LaB::hi(w[i]);
      }
    }
    out[p] = uint4{w[0], w[1], w[2], w[3]};
  }
}
template <int N> __device__ __forceinline__ void la_split(const caf4* t, LaFrag* out) {
  const float v[8] = {t[0][0], t[0][1], t[0][2], t[0][3], t[1][0], t[1][1], t[1][2], t[1][3]};
  uint4 w[N];
  la_split<N>(v, w);
#pragma unroll
  for (int p = 0; p < N; ++p) out[p] = ca_frag<HCLSM_BF16>(w[p]);
}

// acc += sum over the planes whose orders add up to at most MOST (what is left out lies below the last plane kept).
template <int NA, int NB, int MOST> __device__ __forceinline__ caf4 la_mma(const LaFrag* a, const LaFrag* b, caf4 acc) {
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
      if (i + j <= MOST) acc = LaB::mma(a[i], b[j], acc);
  return acc;
}

// Rows of one chunk on their way from global memory: eight elements of a row per unit.
template <int DT, int C, int D, int NT> struct LaStage {
  static constexpr int U = (C * (D / 8) + NT - 1) / NT, RAW = LaT<DT>::RAW, NP = LaT<DT>::NP, ESZ = DT == HCLSM_F32 ? 4 : 2;
  using Tile = CaTile<HCLSM_BF16, D>;
  static constexpr int PLANE = C * Tile::STRIDE;
  uint4 raw[U][RAW];

  static __device__ __forceinline__ int row(int u) { return ((int)threadIdx.x + u * NT) / (D / 8); }
  static __device__ __forceinline__ int chunk(int u) { return ((int)threadIdx.x + u * NT) % (D / 8); }

  // base: the first live token of the chunk at column 0; n live tokens, taken backwards where `back`; d columns
  __device__ __forceinline__ void load(const char* base, int64_t sl, int n, int d, bool back) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = row(u), c = chunk(u) * 8;
#pragma unroll
      for (int k = 0; k < RAW; ++k) raw[u][k] = uint4{0, 0, 0, 0};
      if (r < n && c < d) {
        const char* p = base + ((back ? n - 1 - r : r) * sl + c) * ESZ;
#pragma unroll
        for (int k = 0; k < RAW; ++k) raw[u][k] = reinterpret_cast<const uint4*>(p)[k];
      }
    }
  }
  __device__ __forceinline__ void store(char* t) const {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (row(u) >= C) break;
      uint4 w[NP];
      if constexpr (DT == HCLSM_BF16) {
        w[0] = raw[u][0];
      } else {
        float v[8];
        if constexpr (DT == HCLSM_F16) {
          const uint32_t x[4] = {raw[u][0].x, raw[u][0].y, raw[u][0].z, raw[u][0].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) { v[2 * i] = CaT<HCLSM_F16>::lo(x[i]); v[2 * i + 1] = CaT<HCLSM_F16>::hi(x[i]); }
        } else {
          const caf4 a = __builtin_bit_cast(caf4, raw[u][0]), b = __builtin_bit_cast(caf4, raw[u][1]);
#pragma unroll
          for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
        }
        la_split<NP>(v, w);
      }
#pragma unroll
      for (int p = 0; p < NP; ++p) *reinterpret_cast<uint4*>(t + p * PLANE + Tile::off(row(u), chunk(u))) = w[p];
    }
  }
};

// Operand with rows row0 + 4g .. + 3 and row0 + 16 + 4g .. + 3 as contraction, as CaTile::frag_t, and as its free index the
// columns 32 blk + 8 (li / 4) + 4 m + li % 4: the products of m = 0 and 1 leave a lane with columns 32 blk + 8g .. + 7 of
// the state in order, which is how a row's operand holds them.
template <int D> __device__ __forceinline__ LaFrag la_frag_cols(char* t, int row0, int blk, int m, int li, int g) {
  using Tile = CaTile<HCLSM_BF16, D>;
  const int row = row0 + 4 * g + (li >> 2), chunk = 4 * blk + (li & 3), sub = 8 * m;
  const cas4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ca_lds_s4*)(t + Tile::off(row, chunk) + sub));
  const cas4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ca_lds_s4*)(t + Tile::off(row + 16, chunk) + sub));
  typedef short s8 __attribute__((ext_vector_type(8)));
  const s8 r = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  return __builtin_bit_cast(LaFrag, r);
}

// One workgroup: a head of a batch row, XT = 16 NW columns of X (and of the state and the output), one segment of the
// tokens, chunk after chunk.  Wave w owns 16 columns of the state, in registers for the whole segment; the weights of
// pairs (A_r . B_s) a^(r-s) are shared out over the waves and passed through LDS in the order in which the matrix unit
// reads them.  SUM: the state alone, from zero (the sum of a segment).
template <int DT, int DA, int NW, bool SUM>
__global__ void __launch_bounds__(64 * NW) la_kernel(const LaArgs args) {
  constexpr int NT = 64 * NW, XT = 16 * NW, C = la_chunk(DT, DA), KT = C / 16, NS = DA / 16, NP = LaT<DT>::NP, NC = LaT<DT>::NC;
  constexpr int ESZ = DT == HCLSM_F32 ? 4 : 2, MOST = NC - 1;
  constexpr int NF = KT == 4 ? 6 : 2;       // pairs of 16-token tiles at or below the diagonal
  using SA = LaStage<DT, C, DA, NT>;
  using SX = LaStage<DT, C, XT, NT>;
  using TA = CaTile<HCLSM_BF16, DA>;
  using TX = CaTile<HCLSM_BF16, XT>;
  __shared__ __attribute__((aligned(16))) char ta[SUM ? 16 : NP * SA::PLANE];
  __shared__ __attribute__((aligned(16))) char tb[NP * SA::PLANE];
  __shared__ __attribute__((aligned(16))) char tx[NP * SX::PLANE];
  __shared__ uint4 tp[SUM ? 1 : NF * NC * 64];
  __shared__ float pw[C + 1];               // powers of the decay
  __shared__ float em[C + 1];               // a^n - 1

  uint32_t i = blockIdx.x;
  int ji = 0;
  while (ji + 1 < args.njobs && i >= args.first[ji + 1]) ++ji;
  const LaJob& j = args.job[ji];
  i -= args.first[ji];
  const int seg = (int)(i % (uint32_t)args.nseg);
  i /= (uint32_t)args.nseg;
  const int xt = (int)(i % (uint32_t)j.xtiles), unit = (int)(i / (uint32_t)j.xtiles);
  const int b = unit / args.H, h = unit - b * args.H;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, g = lane >> 4;
  const int live = ca_len(args.lens, args.lens64, b, args.L);
  const bool back = j.back != 0;
  const int x0 = xt * XT, xc = x0 + 16 * wave;      // first column of the workgroup, of the wave

  if ((int)threadIdx.x <= C) {
    const float gd = la_log_decay(args.log_decay, h);
    pw[threadIdx.x] = expf(gd * (float)threadIdx.x);
    em[threadIdx.x] = expm1f(gd * (float)threadIdx.x);
  }

  // tokens of this segment (taken backwards: segment 0 is the last)
  const int sa = back ? args.nseg - 1 - seg : seg;
  const int64_t t_begin = args.nseg > 1 ? (int64_t)sa * args.seg_tokens : 0;
  const int64_t t_stop = args.nseg > 1 ? t_begin + args.seg_tokens : args.L;
  const int t_end = (int)(t_stop < args.L ? t_stop : args.L);
  const int first = (int)(t_begin < args.L ? t_begin : args.L);
  const int nch = (t_end - first + C - 1) / C;

  // the state: tile m of 16 rows holds da = 32 (m / 2) + 8g + 4 (m & 1) + r of column xc + li
  caf4 s[NS];
  const int64_t state = (int64_t)j.da * j.dx;
#pragma unroll
  for (int m = 0; m < NS; ++m) {
    s[m] = caf4{0.f, 0.f, 0.f, 0.f};
    if constexpr (!SUM) {
      const float* p = args.nseg > 1 ? j.seg + ((int64_t)unit * args.nseg + seg) * state : j.s0 ? j.s0 + unit * state : nullptr;
      const int64_t sr = args.nseg > 1 ? j.dx : j.s_r, sc = args.nseg > 1 ? 1 : j.s_c;
      if (p != nullptr && xc + li < j.dx) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int d = 32 * (m >> 1) + 8 * g + 4 * (m & 1) + r;
          if (d < j.da) s[m][r] = p[d * sr + (xc + li) * sc];
        }
      }
    }
  }

  const char* pa = j.a.p + (b * j.a.sb + (h / j.a.group) * j.a.sh) * ESZ;
  const char* pb = j.b.p + (b * j.b.sb + (h / j.b.group) * j.b.sh) * ESZ;
  const char* px = j.x.p + (b * j.x.sb + (h / j.x.group) * j.x.sh + x0) * ESZ;
  SA ra, rb;
  SX rx;
  auto tokens = [&](int k, int& t0, int& n) __attribute__((always_inline)) {
    t0 = first + (back ? nch - 1 - k : k) * C;
    const int e = live < t_end ? live : t_end;
    n = e - t0;
    n = n < 0 ? 0 : n > C ? C : n;
  };
  auto load = [&](int k) __attribute__((always_inline)) {
    int t0, n;
    tokens(k, t0, n);
    if constexpr (!SUM) ra.load(pa + t0 * j.a.sl * ESZ, j.a.sl, n, j.da, back);
    rb.load(pb + t0 * j.b.sl * ESZ, j.b.sl, n, j.da, back);
    rx.load(px + t0 * j.x.sl * ESZ, j.x.sl, n, j.dx - x0, back);
  };
  if (nch > 0) load(0);
  for (int k = 0; k < nch; ++k) {
    int t0, n;
    tokens(k, t0, n);
    __syncthreads();      // every wave is done with the chunk before
    if (n > 0) {
      if constexpr (!SUM) ra.store(ta);
      rb.store(tb);
      rx.store(tx);
    }
    __syncthreads();
    if (k + 1 < nch) load(k + 1);

    caf4 y[KT];
    if (!SUM && n > 0) {
      // weights of pairs: tile (s, t) leaves a lane with s = 4g + r of its t = li
#pragma unroll
      for (int f0 = 0; f0 < NF; f0 += NW) {
        const int f = f0 + wave;
        if (f < NF) {
          const int tt = KT == 4 ? (f < 2 ? f : 2 + ((f - 2) >> 1)) : f, sp = KT == 4 && f >= 2 ? (f & 1) : 0;
          caf4 w[2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int ss = 2 * sp + u;
            w[u] = caf4{0.f, 0.f, 0.f, 0.f};
            if (ss <= tt) {
#pragma unroll
              for (int c = 0; c < DA / 32; ++c) {
                LaFrag fb[NP], fa[NP];
#pragma unroll
                for (int p = 0; p < NP; ++p) {
                  fb[p] = TA::frag(tb + p * SA::PLANE, 16 * ss, c, li, g);
                  fa[p] = TA::frag(ta + p * SA::PLANE, 16 * tt, c, li, g);
                }
                w[u] = la_mma<NP, NP, MOST>(fb, fa, w[u]);
              }
              const int gap = 16 * (tt - ss) + li - 4 * g;
#pragma unroll
              for (int r = 0; r < 4; ++r) w[u][r] = gap >= r ? w[u][r] * (j.cp * pw[gap - r]) : 0.f;
            }
          }
          LaFrag fp[NC];
          la_split<NC>(w, fp);
#pragma unroll
          for (int p = 0; p < NC; ++p) tp[(f * NC + p) * 64 + lane] = __builtin_bit_cast(uint4, fp[p]);
        }
      }
    }
    if constexpr (!SUM) __syncthreads();
    if (n > 0) {
      if constexpr (!SUM) {
        // what the state gives: y^T = S^T A^T
#pragma unroll
        for (int t = 0; t < KT; ++t) y[t] = caf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < DA / 32; ++c) {
          LaFrag fs[NC];
          la_split<NC>(&s[2 * c], fs);
#pragma unroll
          for (int t = 0; t < KT; ++t) {
            LaFrag fa[NP];
#pragma unroll
            for (int p = 0; p < NP; ++p) fa[p] = TA::frag(ta + p * SA::PLANE, 16 * t, c, li, g);
            y[t] = la_mma<NC, NP, MOST>(fs, fa, y[t]);
          }
        }
#pragma unroll
        for (int t = 0; t < KT; ++t) y[t] *= j.ci * pw[16 * t + li + 1 - j.shift];
      }
      LaFrag fx[KT / 2][NP];
#pragma unroll
      for (int sp = 0; sp < KT / 2; ++sp)
#pragma unroll
        for (int p = 0; p < NP; ++p) fx[sp][p] = TX::frag_t(tx + p * SX::PLANE, 32 * sp, wave, li, g);
      if constexpr (!SUM) {
#pragma unroll
        for (int f = 0; f < NF; ++f) {
          const int tt = KT == 4 ? (f < 2 ? f : 2 + ((f - 2) >> 1)) : f, sp = KT == 4 && f >= 2 ? (f & 1) : 0;
          LaFrag fp[NC];
#pragma unroll
          for (int p = 0; p < NC; ++p) fp[p] = ca_frag<HCLSM_BF16>(tp[(f * NC + p) * 64 + lane]);
          y[tt] = la_mma<NP, NC, MOST>(fx[sp], fp, y[tt]);
        }
      }
      // the state behind the chunk
      const float an = pw[n], less = em[n];
#pragma unroll
      for (int m = 0; m < NS; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[m][r] = la_decayed(s[m][r], an, less);
#pragma unroll
      for (int sp = 0; sp < KT / 2; ++sp) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int q = 32 * sp + 16 * (e >> 2) + 4 * g + (e & 3);
          float x = 0.f;
#pragma unroll
          for (int p = NP - 1; p >= 0; --p) x += (float)fx[sp][p][e];
          v[e] = q < n ? x * (j.cu * pw[n - 1 - q + j.shift]) : 0.f;
        }
        uint4 w[3];
        la_split<3>(v, w);
        LaFrag fw[3];
#pragma unroll
        for (int p = 0; p < 3; ++p) fw[p] = ca_frag<HCLSM_BF16>(w[p]);
#pragma unroll
        for (int m = 0; m < NS; ++m) {
          LaFrag fb[NP];
#pragma unroll
          for (int p = 0; p < NP; ++p) fb[p] = la_frag_cols<DA>(tb + p * SA::PLANE, 32 * sp, m >> 1, m & 1, li, g);
          s[m] = la_mma<NP, 3, 2>(fb, fw, s[m]);
        }
      }
    } else if constexpr (!SUM) {
#pragma unroll
      for (int t = 0; t < KT; ++t) y[t] = caf4{0.f, 0.f, 0.f, 0.f};
    }
    if constexpr (!SUM) {
      const int col = xc + 4 * g;
      if (j.y != nullptr && col < j.dx) {
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          const int r = 16 * t + li;
          const int64_t tok = t0 + (r < n && back ? n - 1 - r : r);      // tokens that are not live get zeros
          if (tok < t_end) {
            const int64_t o = ((b * (int64_t)args.L + tok) * args.H + h) * j.dx + col;
            const caf4 v = r < n ? y[t] : caf4{0.f, 0.f, 0.f, 0.f};
            if (j.y32) *reinterpret_cast<caf4*>(j.y + o * 4) = v;
            else ca_store4<DT>(j.y, o, v);
          }
        }
      }
    }
  }

  float* out = SUM ? j.seg + ((int64_t)unit * args.nseg + seg) * state : args.nseg == 1 && j.s1 ? j.s1 + unit * state : nullptr;
  if (out != nullptr && xc + li < j.dx) {
    const int64_t sr = SUM ? j.dx : j.s_r, sc = SUM ? 1 : j.s_c;
#pragma unroll
    for (int m = 0; m < NS; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = 32 * (m >> 1) + 8 * g + 4 * (m & 1) + r;
        if (d < j.da) out[d * sr + (xc + li) * sc] = s[m][r];
      }
  }
}

template <int DT, int DA, int NW>
int la_launch_one(const LaArgs& a, bool sum, hipStream_t st) {
  const dim3 grid(a.first[a.njobs]), block(64 * NW);
  if (sum) hipLaunchKernelGGL((la_kernel<DT, DA, NW, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((la_kernel<DT, DA, NW, false>), grid, block, 0, st, a);
  HCLSM_LAUNCH_CHECK();
  return 0;
}

template <int DT> int la_launch(const LaArgs& a, int da, int xt, bool sum, hipStream_t st) {
  if (xt == 64) {
    if (da == 64) return la_launch_one<DT, 64, 4>(a, sum, st);
    if (da == 128) return la_launch_one<DT, 128, 4>(a, sum, st);
    return la_launch_one<DT, 256, 4>(a, sum, st);
  }
  if (da == 64) return la_launch_one<DT, 64, 8>(a, sum, st);
  if (da == 128) return la_launch_one<DT, 128, 8>(a, sum, st);
  return la_launch_one<DT, 256, 8>(a, sum, st);
}

}  // namespace hclsm
