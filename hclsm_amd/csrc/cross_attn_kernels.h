// Cross-attention kernels, instantiated for one element type per source file (cross_attn_{f32,bf16,f16}.hip).
#pragma once

#include "cross_attn_few.h"

namespace hclsm {

// Two LDS objects of their own, and loops that name them in turn: a read of the one then does not wait for transfers to
// the other (with one object, or an index into two, the compiler has every LDS read wait for all transfers).
#define CA_TWO_BUFFERS(bytes)                                       \
  __shared__ __attribute__((aligned(16))) char buf0[bytes];         \
  __shared__ __attribute__((aligned(16))) char buf1[bytes]

// Bits of the live keys among t0 .. t0 + ROWS - 1: below `end` and not flagged.  p: this lane's flag.
template <int ROWS> __device__ __forceinline__ uint64_t ca_live(int t0, int end, uint8_t p) {
  const int lane = threadIdx.x & 63;
  return __ballot(lane < ROWS && t0 + lane < end && p == 0);
}
template <int ROWS> __device__ __forceinline__ uint8_t ca_flag(const uint8_t* pad, int t0, int end) {
  const int lane = threadIdx.x & 63;
  return pad != nullptr && lane < ROWS && t0 + lane < end ? pad[t0 + lane] : (uint8_t)0;
}
template <int ROWS> constexpr uint64_t CA_FULL = ROWS == 64 ? ~0ull : (1ull << (ROWS & 63)) - 1;

// ---------------------------------------------------------------------------------------------------- forward
//
// NW waves of 16 QT rows each over tiles of KR keys in LDS (two buffers, one barrier per tile), with the running
// maximum and sum of the softmax per row.  Statistics and accumulators are float32; the weights are rounded to the
// operand type (PARTS operands, 2 for few keys) for the second product (half a step, 2^-8 of the value for bf16 and 2^-11
// for fp16; the matrix unit has no wider operand at this rate), their sum is not: the log-sum that the backward reads is
// the float32 one.
//
// What bounds it: the exponentials and the matrix unit together.  Heads of 64 need 512 matrix cycles and about 650 of
// the vector unit (a multiply-add, an exponential, an addition, half a conversion and half a maximum per score) for a
// wave's tile; counted on 8 x 2048 queries, 4099 keys, 12 heads of 64: matrix unit busy 35% of the cycles, vector unit 65%, LDS
// without conflicts 17%.  What was measured to have the one run under the other, and not kept: step u's exponentials
// next to step u + 1's scores in one wave; two halves of a workgroup that a barrier keeps in opposite phases (19 to 45%
// slower); raised priorities around the products or for every other wave; 8 waves to a workgroup; 16 or 48 rows to a
// wave.  Two or three tiles on their way instead of one change nothing (heads of 64: 144 and 143 us; of 128 with tiles of
// 64 keys: 118 both; with tiles of 32, which leave room for three, 137), so the transfers are not what it waits for.
// Measured (bf16): 176 to 182 us there (0.77 PFLOP/s over the live keys); 8 x 2048 queries, 4096 keys, 12 heads of 128: 394 us
// (1.05 PFLOP/s); 8 x 1024, 2048 keys, 12 heads of 128 on 4: 105 us (0.98), matrix unit 36%, vector unit 41% of the
// cycles with 1.46 waves per SIMD on average of the 2 that fit (768 workgroups on 512 places: the last round is half full).
// A matrix product of 8192^3 by the library reaches 1.23 to 1.27 PFLOP/s on the same cards.  Float32, 2 x 1024 queries, 2048
// keys, 12 heads of 64: 142 us with the join of two splits (91 TFLOP/s of the library's 154), of 128: 264 (98), of 256: 654 (79).
template <int DT, int DH, int NW, int QT, int KR, int PARTS>
__global__ void __launch_bounds__(64 * NW) ca_fwd_kernel(const CaArgs a) {
  using A = CaT<DT>;
  using Tile = CaTile<DT, DH>;
  using Frag = typename A::Frag;
  constexpr int NT = 64 * NW, KT = KR / 16, NC = DH / A::KS, ND = DH / 16, NPT = A::NPT, ESZ = (int)sizeof(typename A::T);
  using Stage = CaStage<DT, DH, NT, KR>;
  constexpr int TB = Stage::BYTES;
  CA_TWO_BUFFERS(2 * TB);      // K tile, V tile

  CaWork w;
  if (!ca_work(a, w)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, g = lane >> 4;
  const int row0 = (w.tile * NW + wave) * 16 * QT;
  int k0, k1;
  ca_range(w.keys, a.nsplit, w.split, KR, k0, k1);
  if (w.tile * NW * 16 * QT >= w.rows) k1 = k0;      // no live row in this workgroup

  const char* kp = a.k + (w.b * a.ksb + w.hk * a.ksh) * ESZ;
  const char* vp = a.v + (w.b * a.vsb + w.hk * a.vsh) * ESZ;
  const uint8_t* pad = a.pad ? a.pad + w.b * a.psb : nullptr;

  Frag q[QT][NC];
  {
    const char* qp = a.q + (w.b * a.qsb + (int64_t)w.hk * a.G * a.qsh) * ESZ;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const int r = row0 + 16 * t + li;
      int qi, hg;
      ca_row(a, r < w.rows ? r : 0, qi, hg);
      uint4 f[NC];
      ca_row_frags<DT, DH>(qp + (qi * a.qsl + hg * a.qsh) * ESZ, g, a.dh, r < w.rows, f);
#pragma unroll
      for (int c = 0; c < NC; ++c) q[t][c] = ca_frag<DT>(f[c]);
    }
  }

  caf4 o[QT][ND];
  float m[QT], l[QT];           // reference of the exponentials (log2); sum over this lane's keys
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    m[t] = CA_LOW;
    l[t] = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d) o[t][d] = caf4{0.f, 0.f, 0.f, 0.f};
  }

  const int nt = (k1 - k0 + KR - 1) / KR;
  Stage sk, sv;
  sk.init(a.ksl, a.dh);
  sv.init(a.vsl, a.dh);
  uint8_t flag = 0;
  auto load = [&](int i, char* buf) __attribute__((always_inline)) {
    const int t0 = k0 + i * KR;
    sk.load(kp + t0 * a.ksl * ESZ, k1 - t0, buf, wave);
    sv.load(vp + t0 * a.vsl * ESZ, k1 - t0, buf + TB, wave);
    flag = ca_flag<KR>(pad, t0, k1);
  };
  if (nt > 0) load(0, buf0);
  auto tile = [&](int i, char* tk, char* next) __attribute__((always_inline)) {
    char* tv = tk + TB;
    ca_wait_vmem();
    const uint64_t now = ca_live<KR>(k0 + i * KR, k1, flag);
    __syncthreads();      // tile i is in LDS, and every wave is done with the other buffer
    if (pad != nullptr && now != CA_FULL<KR>) {
      Stage::drop(tk, now);
      Stage::drop(tv, now);
      __syncthreads();
    }
    if (i + 1 < nt) load(i + 1, next);

    caf4 s[QT][KT];
    Frag f[2][NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) f[0][c] = Tile::frag(tk, 0, c, li, g);
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      if (k + 1 < KT) {
#pragma unroll
        for (int c = 0; c < NC; ++c) f[(k + 1) & 1][c] = Tile::frag(tk, 16 * (k + 1), c, li, g);
      }
      ca_fence();
#pragma unroll
      for (int t = 0; t < QT; ++t) s[t][k] = caf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int t = 0; t < QT; ++t) s[t][k] = A::mma(f[k & 1][c], q[t][c], s[t][k]);
      ca_fence();
    }
    // operands of the second product, CV at a time, the first ones on their way during the softmax
    constexpr int J = KT / NPT * ND, CV = J % 4 == 0 ? 4 : 2;
    static_assert(J % CV == 0, "whole groups");
    Frag fv[2][CV];
    auto get_v = [&](int c, Frag* d) {
#pragma unroll
      for (int j = 0; j < CV; ++j)
        d[j] = Tile::frag_t(tv, 16 * NPT * ((c * CV + j) / ND), (c * CV + j) % ND, li, g);
    };
    get_v(0, fv[0]);
    ca_fence();
    if (now != CA_FULL<KR>) {
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        const uint32_t bits = (uint32_t)(now >> (16 * k + 4 * g));
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[t][k][r] = bits >> r & 1 ? s[t][k][r] : -INFINITY;
      }
    }
    // The reference of a row's exponentials follows its maximum only when it falls more than CA_SLACK behind: weights
    // then stay below 2^CA_SLACK, which float32 sums and either 16-bit type hold as exactly as weights below one, and the
    // accumulators are hardly ever rescaled.
    float top[QT];
    bool grew = false;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      float mx = s[t][0][0];
#pragma unroll
      for (int k = 0; k < KT; ++k)
#pragma unroll
        for (int r = 0; r < 4; r += 2) mx = ca_max3(mx, s[t][k][r], s[t][k][r + 1]);
      top[t] = ca_rows4_max(mx) * a.scale_log2;
      grew |= !(top[t] <= m[t] + CA_SLACK<DT>);
    }
    if (__any(grew)) {
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const float to = top[t] <= m[t] + CA_SLACK<DT> ? m[t] : top[t] - CA_BELOW<DT>;
        const float alpha = fast_exp2(m[t] - to);
        m[t] = to;
        l[t] *= alpha;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[t][d] *= alpha;
      }
    }
    Frag p[QT][KT / NPT][PARTS];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
#pragma unroll
      for (int k = 0; k < KT; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[t][k][r] = fast_exp2(s[t][k][r] * a.scale_log2 - m[t]);
      float sum[4] = {l[t], 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KT; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) sum[r] += s[t][k][r];
      l[t] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
      for (int u = 0; u < KT / NPT; ++u) ca_pack_parts<DT, PARTS>(&s[t][u * NPT], p[t][u]);
    }
#pragma unroll
    for (int c = 0; c < J / CV; ++c) {
      if (c + 1 < J / CV) get_v(c + 1, fv[(c + 1) & 1]);
      ca_fence();
#pragma unroll
      for (int j = 0; j < CV; ++j)
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
          for (int e = 0; e < PARTS; ++e)
            o[t][(c * CV + j) % ND] = A::mma(fv[c & 1][j], p[t][(c * CV + j) / ND][e], o[t][(c * CV + j) % ND]);
      ca_fence();
    }
  };
  for (int i = 0; i < nt; i += 2) {
    tile(i, buf0, buf1);
    if (i + 1 < nt) tile(i + 1, buf1, buf0);
  }

  // rows without a live key have l = 0: zeros, and a log-sum of -inf
  const int all = a.Lq * a.G;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const float sum = rows4_sum(l[t]);
    const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    const int r = row0 + 16 * t + li;
    if (r >= all) continue;
    const bool in = r < w.rows;
    int qi, hg;
    ca_row(a, r, qi, hg);
    const int h = w.hk * a.G + hg;
    const float ls2 = in && sum > 0.f ? m[t] + __log2f(sum) : in && sum != sum ? sum : -INFINITY;
    if (a.nsplit > 1) {
      const int64_t pr = ((int64_t)w.split * a.units + w.unit) * all + r;
      if (g == 0) a.part_lse[pr] = ls2;
#pragma unroll
      for (int d = 0; d < ND; ++d)
        if (16 * d + 4 * g < a.dh)
          *reinterpret_cast<caf4*>(a.part + pr * a.dh + 16 * d + 4 * g) = in ? o[t][d] * inv : caf4{0.f, 0.f, 0.f, 0.f};
    } else {
      if (g == 0 && a.lse) a.lse[(w.b * a.Hk * a.G + h) * a.Lq + qi] = ls2 * HCLSM_LN2;
      const int64_t ob = ((w.b * a.Lq + qi) * a.Hk * a.G + h) * (int64_t)a.dh;
#pragma unroll
      for (int d = 0; d < ND; ++d)
        if (16 * d + 4 * g < a.dh) ca_store_out<DT>(a, ob + 16 * d + 4 * g, in ? o[t][d] * inv : caf4{0.f, 0.f, 0.f, 0.f});
    }
  }
}

// ---------------------------------------------------------------------------------------- gradient of the queries
//
// As the forward, with S^T and dP^T = V g^T formed per tile, p = exp(s - lse), ds = p (dP - delta) and
// dQ^T = K^T ds^T.  delta = sum(g o) per row is formed here and left for the second kernel.  ds is rounded to the
// operand type for its product, as the weights are in the forward (float16: at a power of two of its own, CA_RANGED).
// Three products, two of which the kernel for dk and dv forms again: that costs two products in seven, and leaves no sum
// of dq over key tiles to atomics.  Measured: 8 x 1024 queries, 2048 keys, 12 heads of 128 on 4, bf16: 174 us, 0.89 PFLOP/s;
// matrix unit busy 34% of the cycles, vector unit 29%, 0.92 waves per SIMD of the one that its registers leave (three whole
// rounds): in what is left that wave waits, hardly for LDS (2% of its time).  Float32, 2 x 1024, 2048 keys, 12 heads of 64: 199
// us (97 TFLOP/s), of 128: 400 (97).
template <int DT, int DH, int NW, int QT, int KR, bool PIPE, int PARTS>
__global__ void __launch_bounds__(64 * NW) ca_dq_kernel(const CaArgs a) {
  using A = CaT<DT>;
  using Tile = CaTile<DT, DH>;
  using Frag = typename A::Frag;
  constexpr int NT = 64 * NW, KT = KR / 16, NC = DH / A::KS, ND = DH / 16, NPT = A::NPT, ESZ = (int)sizeof(typename A::T);
  using Stage = CaStage<DT, DH, NT, KR>;
  constexpr int TB = Stage::BYTES;
  CA_TWO_BUFFERS(2 * TB);      // K tile, V tile

  CaWork w;
  if (!ca_work(a, w)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, g = lane >> 4;
  const int row0 = (w.tile * NW + wave) * 16 * QT;
  int k0, k1;
  ca_range(w.keys, a.nsplit, w.split, KR, k0, k1);
  if (w.tile * NW * 16 * QT >= w.rows || a.dq == nullptr) k1 = k0;      // (dq not wanted: delta alone)

  const char* kp = a.k + (w.b * a.ksb + w.hk * a.ksh) * ESZ;
  const char* vp = a.v + (w.b * a.vsb + w.hk * a.vsh) * ESZ;
  const uint8_t* pad = a.pad ? a.pad + w.b * a.psb : nullptr;

  Frag q[QT][NC], go[QT][NC];
  float lse2[QT];
  caf4 ndelta[QT];      // -delta of the lane's row: the accumulator that dP starts from
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = row0 + 16 * t + li;
    const bool in = r < w.rows;
    int qi, hg;
    ca_row(a, in ? r : 0, qi, hg);
    const int h = w.hk * a.G + hg;
    const int64_t stat = (w.b * a.Hk * a.G + h) * a.Lq + qi;
    uint4 fq[NC], fg[NC], fo[NC];
    ca_row_frags<DT, DH>(a.q + (w.b * a.qsb + qi * a.qsl + h * a.qsh) * ESZ, g, a.dh, in, fq);
    ca_row_frags<DT, DH>(a.g + (w.b * a.gsb + qi * a.gsl + h * a.gsh) * ESZ, g, a.dh, in, fg);
    ca_row_frags<DT, DH>(a.o + ((w.b * a.Lq + qi) * a.Hk * a.G + h) * (int64_t)a.dh * ESZ, g, a.dh, in, fo);
    uint4 fl[NC];
    const bool lo = a.olo != nullptr;
    ca_row_frags<DT, DH>(a.olo + ((w.b * a.Lq + qi) * a.Hk * a.G + h) * (int64_t)a.dh * ESZ, g, a.dh, in && lo, fl);
    const float ls = in ? a.lse[stat] : -INFINITY;
    lse2[t] = ls == -INFINITY ? INFINITY : ls * HCLSM_LOG2E;      // no key: every weight is exp(-inf)
    float dsum = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      dsum = ca_dot<DT>(fg[c], fo[c], dsum);
      dsum = ca_dot<DT>(fg[c], fl[c], dsum);
      q[t][c] = ca_frag<DT>(fq[c]);
      go[t][c] = ca_frag<DT>(fg[c]);
    }
    dsum = rows4_sum(dsum);
    ndelta[t] = caf4{-dsum, -dsum, -dsum, -dsum};
    if (in && g == 0 && w.split == 0) a.delta[stat] = dsum;
  }

  caf4 dq[QT][ND];
  float up[QT];         // float16: factor of the row's ds
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    up[t] = ca_pow2(CA_F16_START);
#pragma unroll
    for (int d = 0; d < ND; ++d) dq[t][d] = caf4{0.f, 0.f, 0.f, 0.f};
  }

  const int nt = (k1 - k0 + KR - 1) / KR;
  Stage sk, sv;
  sk.init(a.ksl, a.dh);
  sv.init(a.vsl, a.dh);
  uint8_t flag = 0;
  auto load = [&](int i, char* buf) __attribute__((always_inline)) {
    const int t0 = k0 + i * KR;
    sk.load(kp + t0 * a.ksl * ESZ, k1 - t0, buf, wave);
    sv.load(vp + t0 * a.vsl * ESZ, k1 - t0, buf + TB, wave);
    flag = ca_flag<KR>(pad, t0, k1);
  };
  if (nt > 0) load(0, buf0);
  auto tile = [&](int i, char* tk, char* next) __attribute__((always_inline)) {
    char* tv = tk + TB;
    ca_wait_vmem();
    const uint64_t now = ca_live<KR>(k0 + i * KR, k1, flag);
    __syncthreads();      // tile i is in LDS, and every wave is done with the other buffer
    if (pad != nullptr && now != CA_FULL<KR>) {
      Stage::drop(tk, now);
      Stage::drop(tv, now);
      __syncthreads();
    }
    if (i + 1 < nt) load(i + 1, next);
    constexpr int U = KT / NPT;
    caf4 s[2][QT][NPT], dp[2][QT][NPT];
    // S^T and dP^T of step u (16 NPT keys): operands of a 16-key tile are read while the tile before is multiplied
    auto scores = [&](int u, caf4 (*s)[NPT], caf4 (*dp)[NPT]) __attribute__((always_inline)) {
      Frag fk[2][NC], fv[2][NC];
      auto get = [&](int k, int b) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          fk[b][c] = Tile::frag(tk, 16 * (u * NPT + k), c, li, g);
          fv[b][c] = Tile::frag(tv, 16 * (u * NPT + k), c, li, g);
        }
      };
      get(0, 0);
#pragma unroll
      for (int k = 0; k < NPT; ++k) {
        if (k + 1 < NPT) get(k + 1, (k + 1) & 1);
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          s[t][k] = caf4{0.f, 0.f, 0.f, 0.f};
          dp[t][k] = ndelta[t];
        }
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int t = 0; t < QT; ++t) {
            s[t][k] = A::mma(fk[k & 1][c], q[t][c], s[t][k]);
            dp[t][k] = A::mma(fv[k & 1][c], go[t][c], dp[t][k]);
          }
      }
    };
    if (PIPE) scores(0, s[0], dp[0]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      ca_fence();
      if (!PIPE) scores(u, s[u & 1], dp[u & 1]);
      else if (u + 1 < U) scores(u + 1, s[(u + 1) & 1], dp[(u + 1) & 1]);      // the vector unit works on step u meanwhile
      Frag ds[QT][PARTS];
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int k = 0; k < NPT; ++k)
#pragma unroll
          for (int r = 0; r < 4; ++r) dp[u & 1][t][k][r] *= fast_exp2(s[u & 1][t][k][r] * a.scale_log2 - lse2[t]);
      if (now != CA_FULL<KR>) {
#pragma unroll
        for (int k = 0; k < NPT; ++k) {
          const uint32_t bits = (uint32_t)(now >> (16 * (u * NPT + k) + 4 * g));
#pragma unroll
          for (int t = 0; t < QT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) dp[u & 1][t][k][r] = bits >> r & 1 ? dp[u & 1][t][k][r] : 0.f;
        }
      }
      if constexpr (CA_RANGED<DT>) {
        float most[QT];
        bool past = false;
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          most[t] = ca_scale_most<NPT>(dp[u & 1][t], up[t]);
          past |= most[t] > CA_F16_MOST;
        }
        if (__any(past)) {
#pragma unroll
          for (int t = 0; t < QT; ++t) {
            const float f = ca_lowered(ca_rows4_max(most[t]));
            up[t] *= f;
#pragma unroll
            for (int k = 0; k < NPT; ++k) dp[u & 1][t][k] *= f;
#pragma unroll
            for (int d = 0; d < ND; ++d) dq[t][d] *= f;
          }
        }
      }
#pragma unroll
      for (int t = 0; t < QT; ++t) ca_pack_parts<DT, PARTS>(dp[u & 1][t], ds[t]);
      constexpr int CV = ND < 4 ? ND : ND % 4 == 0 ? 4 : 2;
      Frag ft[2][CV];
      auto get_t = [&](int c, int b) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < CV; ++j) ft[b][j] = Tile::frag_t(tk, 16 * NPT * u, c * CV + j, li, g);
      };
      get_t(0, 0);
      ca_fence();
#pragma unroll
      for (int c = 0; c < ND / CV; ++c) {
        if (c + 1 < ND / CV) get_t(c + 1, (c + 1) & 1);
        ca_fence();
#pragma unroll
        for (int j = 0; j < CV; ++j)
#pragma unroll
          for (int t = 0; t < QT; ++t)
#pragma unroll
            for (int e = 0; e < PARTS; ++e) dq[t][c * CV + j] = A::mma(ft[c & 1][j], ds[t][e], dq[t][c * CV + j]);
        ca_fence();
      }
    }
  };
  for (int i = 0; i < nt; i += 2) {
    tile(i, buf0, buf1);
    if (i + 1 < nt) tile(i + 1, buf1, buf0);
  }

  if (a.dq == nullptr) return;
  const int all = a.Lq * a.G;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = row0 + 16 * t + li;
    if (r >= all) continue;
    const bool in = r < w.rows;
    int qi, hg;
    ca_row(a, r, qi, hg);
    const int64_t ob = a.nsplit > 1 ? (((int64_t)w.split * a.units + w.unit) * all + r) * a.dh
                                    : ((w.b * a.Lq + qi) * a.Hk * a.G + w.hk * a.G + hg) * (int64_t)a.dh;
    if constexpr (CA_RANGED<DT>) {
#pragma unroll
      for (int d = 0; d < ND; ++d) dq[t][d] *= ca_unscaled(up[t]);
    }
#pragma unroll
    for (int d = 0; d < ND; ++d)
      if (16 * d + 4 * g < a.dh) {
        const caf4 v = in ? dq[t][d] * a.scale : caf4{0.f, 0.f, 0.f, 0.f};
        if (a.nsplit > 1) *reinterpret_cast<caf4*>(a.part + ob + 16 * d + 4 * g) = v;
        else ca_store4<DT>(a.dq, ob + 16 * d + 4 * g, v);
      }
  }
}

// ------------------------------------------------------------------------------- gradients of the keys and values
//
// NW waves of 16 KT keys each, K and V operands in registers, over tiles of RR rows (q and g in LDS):
// S = Q K^T and dP = g V^T with a lane per key, then dV^T = g^T p and dK^T = Q^T ds.  Shared heads are rows of the
// unit, so their gradients are added here.  Keys that are not live get zeros.
// Four products.  Measured on the sizes above: 389 us with dq, so 215 of its own, 0.96 PFLOP/s; matrix unit busy 37% of the
// cycles, vector unit 31%, one wave per SIMD, which waits for the rest as in ca_dq_kernel (the accumulators and operands of 32
// keys of 128 take 300 registers; 16 keys per wave and two waves per SIMD measured the same).  Float32: 266 us (97 TFLOP/s)
// and 430 (120).
template <int DT, int DH, int NW, int KT, int RR, bool PIPE, int PARTS>
__global__ void __launch_bounds__(64 * NW) ca_dkv_kernel(const CaArgs a) {
  using A = CaT<DT>;
  using Tile = CaTile<DT, DH>;
  using Frag = typename A::Frag;
  constexpr int NT = 64 * NW, RT = RR / 16, NC = DH / A::KS, ND = DH / 16, NPT = A::NPT, ESZ = (int)sizeof(typename A::T);
  using Stage = CaStage<DT, DH, NT, RR>;
  constexpr int TB = Stage::BYTES, BUF = 2 * TB + RR * 8;
  CA_TWO_BUFFERS(BUF);         // Q tile, g tile, RR log-sums, RR negated deltas

  CaWork w;
  if (!ca_work(a, w)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, g = lane >> 4;
  const int key0 = (w.tile * NW + wave) * 16 * KT;
  const int step = ca_row_step(a.G, RR);      // rows of a tile: whole queries
  int r0, r1;
  ca_range(w.rows, a.nsplit, w.split, step, r0, r1);
  if (w.tile * NW * 16 * KT >= w.keys) r1 = r0;

  const char* kp = a.k + (w.b * a.ksb + w.hk * a.ksh) * ESZ;
  const char* vp = a.v + (w.b * a.vsb + w.hk * a.vsh) * ESZ;
  const char* qp = a.q + (w.b * a.qsb + (int64_t)w.hk * a.G * a.qsh) * ESZ;
  const char* gp = a.g + (w.b * a.gsb + (int64_t)w.hk * a.G * a.gsh) * ESZ;
  const int64_t stat0 = (w.b * a.Hk + w.hk) * a.G * (int64_t)a.Lq;

  Frag fk[KT][NC], fv[KT][NC];
  bool live[KT];
#pragma unroll
  for (int t = 0; t < KT; ++t) {
    const int key = key0 + 16 * t + li;
    live[t] = key < w.keys && (a.pad == nullptr || a.pad[w.b * a.psb + key] == 0);
    const int kk = live[t] ? key : 0;
    uint4 f0[NC], f1[NC];
    ca_row_frags<DT, DH>(kp + kk * a.ksl * ESZ, g, a.dh, live[t], f0);
    ca_row_frags<DT, DH>(vp + kk * a.vsl * ESZ, g, a.dh, live[t], f1);
#pragma unroll
    for (int c = 0; c < NC; ++c) { fk[t][c] = ca_frag<DT>(f0[c]); fv[t][c] = ca_frag<DT>(f1[c]); }
  }
  caf4 dk[KT][ND], dv[KT][ND];
  float up[KT];         // float16: factor of the key's ds, formed from weights that have one of 2^12 already
#pragma unroll
  for (int t = 0; t < KT; ++t) {
    up[t] = ca_pow2(CA_F16_START) * CA_P_DOWN<DT>;
#pragma unroll
    for (int d = 0; d < ND; ++d) dk[t][d] = dv[t][d] = caf4{0.f, 0.f, 0.f, 0.f};
  }

  const int nt = (r1 - r0 + step - 1) / step;
  Stage sq, sg;
  float st_lse = -INFINITY, st_delta = 0.f;
  int st_q = 0, st_h = 0;
  auto init = [&](int phase) {
    sq.init_rows(a, a.qsl, a.qsh, phase, step);
    sg.init_rows(a, a.gsl, a.gsh, phase, step);
    ca_row(a, phase + (int)threadIdx.x, st_q, st_h);
  };
  init(0);
  auto load = [&](int i, char* buf) __attribute__((always_inline)) {
    const int t0 = r0 + i * step;
    int q0, phase;
    ca_row(a, t0, q0, phase);
    if (a.G > RR) init(phase);       // more heads to a query than rows to a tile: tiles begin inside a query
    const int n = r1 - t0 < step ? r1 - t0 : RR;
    sq.load(qp + q0 * a.qsl * ESZ, n, buf, wave);
    sg.load(gp + q0 * a.gsl * ESZ, n, buf + TB, wave);
    st_lse = -INFINITY;
    st_delta = 0.f;
    if ((int)threadIdx.x < step && t0 + (int)threadIdx.x < r1) {
      const int64_t j = stat0 + (int64_t)st_h * a.Lq + q0 + st_q;
      st_lse = a.lse[j];          // looked at when the tile's turn comes: here it would wait for the tile
      st_delta = a.delta[j];
    }
  };
  if (nt > 0) load(0, buf0);
  auto tile = [&](int i, char* tq, char* next) __attribute__((always_inline)) {
    char* tg = tq + TB;
    float* stat = reinterpret_cast<float*>(tq + 2 * TB);
    if ((int)threadIdx.x < RR) {       // rows past the last one, and rows without keys: every weight is exp(-inf)
      stat[threadIdx.x] = st_lse == -INFINITY ? INFINITY : st_lse * HCLSM_LOG2E - CA_P_SHIFT<DT>;
      stat[RR + threadIdx.x] = -st_delta;
    }
    ca_wait_vmem();
    __syncthreads();
    if (i + 1 < nt) load(i + 1, next);
    constexpr int U = RT / NPT;
    caf4 s[2][KT][NPT], dp[2][KT][NPT];
    // S and dP of step u (16 NPT rows): operands of a 16-row tile are read while the tile before is multiplied
    auto scores = [&](int u, caf4 (*s)[NPT], caf4 (*dp)[NPT]) __attribute__((always_inline)) {
      Frag fq[2][NC], fg[2][NC];
      auto get = [&](int k, int b) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          fq[b][c] = Tile::frag(tq, 16 * (u * NPT + k), c, li, g);
          fg[b][c] = Tile::frag(tg, 16 * (u * NPT + k), c, li, g);
        }
      };
      get(0, 0);
#pragma unroll
      for (int k = 0; k < NPT; ++k) {
        if (k + 1 < NPT) get(k + 1, (k + 1) & 1);
        const caf4 nd = *reinterpret_cast<const caf4*>(stat + RR + 16 * (u * NPT + k) + 4 * g);      // -delta
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          s[t][k] = caf4{0.f, 0.f, 0.f, 0.f};
          dp[t][k] = nd;
        }
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int t = 0; t < KT; ++t) {
            s[t][k] = A::mma(fq[k & 1][c], fk[t][c], s[t][k]);
            dp[t][k] = A::mma(fg[k & 1][c], fv[t][c], dp[t][k]);
          }
      }
    };
    if (PIPE) scores(0, s[0], dp[0]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      ca_fence();
      if (!PIPE) scores(u, s[u & 1], dp[u & 1]);
      else if (u + 1 < U) scores(u + 1, s[(u + 1) & 1], dp[(u + 1) & 1]);      // the vector unit works on step u meanwhile
      Frag p[KT][PARTS], ds[KT][PARTS];
#pragma unroll
      for (int k = 0; k < NPT; ++k) {
        const caf4 ls = *reinterpret_cast<const caf4*>(stat + 16 * (u * NPT + k) + 4 * g);
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            s[u & 1][t][k][r] = fast_exp2(s[u & 1][t][k][r] * a.scale_log2 - ls[r]);
            dp[u & 1][t][k][r] *= s[u & 1][t][k][r];
          }
      }
      if constexpr (CA_RANGED<DT>) {
        float most[KT];
        bool past = false;
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          most[t] = ca_scale_most<NPT>(dp[u & 1][t], up[t]);
          past |= live[t] && most[t] > CA_F16_MOST;
        }
        if (__any(past)) {
#pragma unroll
          for (int t = 0; t < KT; ++t) {
            const float f = ca_lowered(ca_rows4_max(most[t]));
            up[t] *= f;
#pragma unroll
            for (int k = 0; k < NPT; ++k) dp[u & 1][t][k] *= f;
#pragma unroll
            for (int d = 0; d < ND; ++d) dk[t][d] *= f;
          }
        }
      }
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        ca_pack_parts<DT, PARTS>(s[u & 1][t], p[t]);
        ca_pack_parts<DT, PARTS>(dp[u & 1][t], ds[t]);
      }
      constexpr int CV = ND < 2 ? ND : 2;
      Frag tg2[2][CV], tq2[2][CV];
      auto get_t = [&](int c, int b) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < CV; ++j) {
          tg2[b][j] = Tile::frag_t(tg, 16 * NPT * u, c * CV + j, li, g);
          tq2[b][j] = Tile::frag_t(tq, 16 * NPT * u, c * CV + j, li, g);
        }
      };
      get_t(0, 0);
      ca_fence();
#pragma unroll
      for (int c = 0; c < ND / CV; ++c) {
        if (c + 1 < ND / CV) get_t(c + 1, (c + 1) & 1);
        ca_fence();
#pragma unroll
        for (int j = 0; j < CV; ++j)
#pragma unroll
          for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int e = 0; e < PARTS; ++e) {
              dv[t][c * CV + j] = A::mma(tg2[c & 1][j], p[t][e], dv[t][c * CV + j]);
              dk[t][c * CV + j] = A::mma(tq2[c & 1][j], ds[t][e], dk[t][c * CV + j]);
            }
        ca_fence();
      }
    }
  };
  for (int i = 0; i < nt; i += 2) {
    tile(i, buf0, buf1);
    if (i + 1 < nt) tile(i + 1, buf1, buf0);
  }

  // Keys that are not live read as zeros: their weights exp(-lse) mean nothing (they may overflow) but stay in the key's
  // own column of either sum, and the rows are written as zeros.
  const int64_t half = (int64_t)a.nsplit * a.units * a.Lk * a.dh;      // split: dk sums, then dv sums
#pragma unroll
  for (int t = 0; t < KT; ++t) {
    const int key = key0 + 16 * t + li;
    if (key >= a.Lk) continue;
    const int64_t ob = a.nsplit > 1 ? (((int64_t)w.split * a.units + w.unit) * a.Lk + key) * a.dh
                                    : ((w.b * a.Lk + key) * a.Hk + w.hk) * (int64_t)a.dh;
    if constexpr (CA_RANGED<DT>) {
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        dk[t][d] *= ca_unscaled(up[t]) * CA_P_DOWN<DT>;
        dv[t][d] *= CA_P_DOWN<DT>;
      }
    }
#pragma unroll
    for (int d = 0; d < ND; ++d)
      if (16 * d + 4 * g < a.dh) {
        const int64_t i = ob + 16 * d + 4 * g;
        const caf4 zero = {0.f, 0.f, 0.f, 0.f}, vk = live[t] ? dk[t][d] * a.scale : zero, vv = live[t] ? dv[t][d] : zero;
        if (a.nsplit > 1) {
          *reinterpret_cast<caf4*>(a.part + i) = vk;
          *reinterpret_cast<caf4*>(a.part + half + i) = vv;
        } else {
          ca_store4<DT>(a.dk, i, vk);
          ca_store4<DT>(a.dv, i, vv);
        }
      }
  }
}

// ------------------------------------------------------------------------------------------------------- launches

// Tile sizes by the bytes of a padded row: two buffers of two tiles have to fit the 160 KB of LDS next to
// another workgroup where rows are short, and the accumulators and operands of a wave its registers.
template <int DT, int DH> struct CaShape {
  static constexpr int RB = DH * (int)sizeof(typename CaT<DT>::T);
  static constexpr int TR = RB <= 256 ? 64 : 32;      // rows of a tile
  static constexpr int T = RB <= 256 ? 2 : 1;         // 16-row tiles per wave
  // Scores of the next step formed while the vector unit works on this one's: a second set of score tiles, which
  // pays where it leaves the same number of waves per SIMD.  Measured on 8 x 1024 queries, 2048 keys, 12 heads, bf16 (us
  // without -> with): dq of heads of 32: 69 -> 66, 64: 103 -> 96, 96: 128 -> 127, 128: 177 -> 181, 192: 301 -> 289, 256: 328
  // -> 356; dk and dv 78 -> 77, 126 -> 122, 211 -> 225, 284 -> 253, 419 -> 389, 637 -> 690; float32 (2 batch rows), heads of
  // 64: 194 -> 194 and 265 -> 266, of 128: 397 -> 394 and 431 -> 460.
  static constexpr bool PIPE_Q = RB <= 256, PIPE_KV = RB <= 256 && DH % 64 == 0;
  static constexpr int FINE = DT == HCLSM_F32 ? 1 : 2;      // operands that hold the weights of few keys
  static_assert(4 * CaTile<DT, DH>::bytes(TR, 256) + 2 * TR * 8 <= 160 * 1024, "two buffers of two tiles");
};

template <int DT> inline bool ca_fine(const CaArgs& a) { return DT != HCLSM_F32 && a.Lk <= CA_FINE_KEYS; }

inline bool ca_by_xcd(int64_t units) { return units % 8 == 0 || units >= 64; }

template <typename K>
int ca_launch(K kernel, CaArgs& a, int64_t batch, int64_t rows, int per_wg, int threads, hipStream_t st) {
  const int64_t units = batch * a.Hk, tiles = (rows + per_wg - 1) / per_wg;
  a.units = (int)units;
  a.tiles = (int)tiles;
  a.by_xcd = ca_by_xcd(units);
  const int64_t blocks = (a.by_xcd ? (units + 7) / 8 * 8 : units) * tiles * a.nsplit;
  if (blocks == 0) return 0;
  if (blocks > 0x7fffffff / threads) return HCLSM_ERR_UNSUPPORTED;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), 0, st, a);
  HCLSM_LAUNCH_CHECK();
  return 0;
}

template <int DT, int DH> int ca_forward_dh(CaArgs& a, int64_t batch, void* ws, int64_t ws_bytes, hipStream_t st) {
  using S = CaShape<DT, DH>;
  const CaPlan p = ca_forward_plan(batch, a.Lq, a.Lk, a.Hk, a.G, a.dh, DT);
  const int64_t rows = (int64_t)a.Lq * a.G;
  a.nsplit = p.nsplit;
  if (p.nsplit > 1) {
    const int64_t n = (int64_t)p.nsplit * batch * a.Hk * rows;
    if (ws == nullptr) return HCLSM_ERR_NULL;
    if (ws_bytes < n * (a.dh + 1) * 4) return HCLSM_ERR_SHAPE;
    a.part = (float*)ws;
    a.part_lse = a.part + n * a.dh;
  }
  int rc = HCLSM_ERR_UNSUPPORTED;
  if (p.few == 1) {
    if constexpr (S::RB <= CA_FEW1_BYTES) rc = ca_launch(ca_few_kernel<DT, DH, 4, 1>, a, batch, rows, 16, 256, st);
  } else if (p.few == 2) {
    if constexpr (S::RB <= ca_few2_bytes(DT)) rc = ca_launch(ca_few_kernel<DT, DH, 4, 2>, a, batch, rows, 32, 256, st);
  } else {
    rc = ca_fine<DT>(a)                      ? ca_launch(ca_fwd_kernel<DT, DH, 4, 1, CA_FINE_KEYS, S::FINE>, a, batch, rows, 64, 256, st)
         : ca_tile_rows(rows, S::RB) == 64 ? ca_launch(ca_fwd_kernel<DT, DH, 4, 1, S::TR, 1>, a, batch, rows, 64, 256, st)
                                           : ca_launch(ca_fwd_kernel<DT, DH, 4, S::T, S::TR, 1>, a, batch, rows, 128, 256, st);
  }
  if (rc || p.nsplit == 1) return rc;
  return ca_join(a, DT, st);
}

template <int DT, int DH> int ca_backward_dh(CaArgs& a, int64_t batch, void* ws, int64_t ws_bytes, hipStream_t st) {
  using S = CaShape<DT, DH>;
  const CaPlan p = ca_backward_plan(batch, a.Lq, a.Lk, a.Hk, a.G, a.dh, DT);
  const int64_t rows = (int64_t)a.Lq * a.G, units = batch * a.Hk;
  if (ws_bytes < ca_backward_bytes(p, batch, a.Lq, a.Lk, a.Hk, a.G, a.dh)) return HCLSM_ERR_SHAPE;
  char* w = (char*)ws;
  a.nsplit = p.nsplit;
  if (p.few) {
    a.part = (float*)w;
    int rc = HCLSM_ERR_UNSUPPORTED;
    if constexpr (S::RB <= CA_FEW_BWD_BYTES) rc = ca_launch(ca_few_bwd_kernel<DT, DH, 4>, a, batch, 1, 1, 256, st);
    return rc || p.nsplit == 1 || a.dq == nullptr ? rc : ca_sum(a, 0, DT, st);
  }
  a.delta = (float*)w;
  w += (units * rows * 4 + 255) / 256 * 256;
  a.part = (float*)w;
  if (a.dq == nullptr) a.nsplit = 1;
  const bool fine = ca_fine<DT>(a);
  if (int rc = fine ? ca_launch(ca_dq_kernel<DT, DH, 4, 1, CA_FINE_KEYS, false, S::FINE>, a, batch, rows, 64, 256, st)
               : ca_tile_rows(rows, S::RB) == 64
                   ? ca_launch(ca_dq_kernel<DT, DH, 4, 1, S::TR, S::PIPE_Q, 1>, a, batch, rows, 64, 256, st)
                   : ca_launch(ca_dq_kernel<DT, DH, 4, S::T, S::TR, S::PIPE_Q, 1>, a, batch, rows, 128, 256, st))
    return rc;
  if (a.nsplit > 1) {
    if (int rc = ca_sum(a, 0, DT, st)) return rc;
    w += a.nsplit * units * rows * a.dh * 4;
  }
  if (a.dk == nullptr) return 0;
  a.nsplit = p.nrows;
  a.part = (float*)w;
  if (int rc = fine ? ca_launch(ca_dkv_kernel<DT, DH, 4, 1, S::TR, false, S::FINE>, a, batch, a.Lk, 64, 256, st)
               : ca_tile_rows(a.Lk, S::RB) == 64
                   ? ca_launch(ca_dkv_kernel<DT, DH, 4, 1, S::TR, S::PIPE_KV, 1>, a, batch, a.Lk, 64, 256, st)
                   : ca_launch(ca_dkv_kernel<DT, DH, 4, S::T, S::TR, S::PIPE_KV, 1>, a, batch, a.Lk, 128, 256, st))
    return rc;
  return p.nrows > 1 ? ca_sum(a, 1, DT, st) : 0;
}

template <int DT> int ca_forward_dt(CaArgs a, int64_t batch, void* ws, int64_t ws_bytes, hipStream_t st) {
  if (a.dh <= 32) return ca_forward_dh<DT, 32>(a, batch, ws, ws_bytes, st);
  if (a.dh <= 64) return ca_forward_dh<DT, 64>(a, batch, ws, ws_bytes, st);
  if (a.dh <= 96) return ca_forward_dh<DT, 96>(a, batch, ws, ws_bytes, st);
  if (a.dh <= 128) return ca_forward_dh<DT, 128>(a, batch, ws, ws_bytes, st);
  if (a.dh <= 192) return ca_forward_dh<DT, 192>(a, batch, ws, ws_bytes, st);
  return ca_forward_dh<DT, 256>(a, batch, ws, ws_bytes, st);
}
template <int DT> int ca_backward_dt(CaArgs a, int64_t batch, void* ws, int64_t ws_bytes, hipStream_t st) {
  if (a.dh <= 32) return ca_backward_dh<DT, 32>(a, batch, ws, ws_bytes, st);
  if (a.dh <= 64) return ca_backward_dh<DT, 64>(a, batch, ws, ws_bytes, st);
  if (a.dh <= 96) return ca_backward_dh<DT, 96>(a, batch, ws, ws_bytes, st);
  if (a.dh <= 128) return ca_backward_dh<DT, 128>(a, batch, ws, ws_bytes, st);
  if (a.dh <= 192) return ca_backward_dh<DT, 192>(a, batch, ws, ws_bytes, st);
  return ca_backward_dh<DT, 256>(a, batch, ws, ws_bytes, st);
}

}  // namespace hclsm
