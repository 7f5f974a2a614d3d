// Cross attention of few rows: at most 32 rows of a unit (one query and its shared heads, or a frame's slots), where
// reading the keys and values is the work.
#pragma once

#include "cross_attn.h"

namespace hclsm {

// Columns of an output tile: the head is cut into groups of 16 W columns (W = 8, 4 or 2), and within a group at column c0 the
// tile nt < W holds columns c0 + W i + nt for its 16 rows i.  A lane then reads its second operand's columns (i = li) as one
// vector of W elements per key, straight from global memory, and holds 4 W consecutive columns of the result.
template <int DT, int DH> struct CaGroups {
  static constexpr int MAXW = DT == HCLSM_F32 ? 4 : 8;
  static constexpr int NT = DH / 16;
  static constexpr int count() {
    int n = 0;
    for (int t = NT; t > 0; ++n) t -= width_of(t);
    return n;
  }
  static constexpr int width_of(int left) { return left >= MAXW ? MAXW : left >= 4 ? 4 : 2; }
  static constexpr int first(int k) {       // first tile of group k
    int t = 0;
    for (int i = 0; i < k; ++i) t += width_of(NT - t);
    return t;
  }
  static constexpr int width(int k) { return width_of(NT - first(k)); }
  static constexpr int N = count();
};

// W elements of 2 or 4 bytes as 32-bit words, in one access
template <int WORDS> __device__ __forceinline__ void ca_load_words(const char* p, uint32_t* w) {
  if constexpr (WORDS == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (WORDS == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// One step's operands of a wave: SK = 16 NPT keys.
template <int DT, int DH> struct CaStep {
  using A = CaT<DT>;
  static constexpr int NPT = A::NPT, NC = DH / A::KS, ESZ = (int)sizeof(typename A::T), SK = 16 * NPT;
  static constexpr int VW = DH / 16 * ESZ / 4;      // words of a key's columns per lane
  uint4 k[NPT][NC];
  uint32_t v[NPT * 4][VW];

  // t0 .. t0 + SK - 1 of the keys; rows past the last one are read at its address
  __device__ __forceinline__ void load(const CaArgs& a, const char* kp, const char* vp, int t0, int last, int li, int g) {
#pragma unroll
    for (int t = 0; t < NPT; ++t) {
      const int row = t0 + 16 * t + li;
      const char* p = kp + (row < last ? row : last) * a.ksl * ESZ;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int e = (4 * c + g) * A::EPC;
        k[t][c] = uint4{0, 0, 0, 0};
        if (e < a.dh) k[t][c] = *reinterpret_cast<const uint4*>(p + e * ESZ);
      }
    }
#pragma unroll
    for (int t = 0; t < NPT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = t0 + 16 * t + 4 * g + r;
        const char* p = vp + (row < last ? row : last) * a.vsl * ESZ;
        load_v<0>(a, p, li, v[4 * t + r]);
      }
  }
  template <int K> __device__ __forceinline__ void load_v(const CaArgs& a, const char* p, int li, uint32_t* w) {
    if constexpr (K < CaGroups<DT, DH>::N) {
      constexpr int F = CaGroups<DT, DH>::first(K), W = CaGroups<DT, DH>::width(K), WORDS = W * ESZ / 4;
      const int col = 16 * F + W * li;
#pragma unroll
      for (int i = 0; i < WORDS; ++i) w[F * ESZ / 4 + i] = 0;
      if (col < a.dh) ca_load_words<WORDS>(p + col * ESZ, w + F * ESZ / 4);
      load_v<K + 1>(a, p, li, w);
    }
  }
  // second operand of tile nt: its column of each of the lane's keys
  __device__ __forceinline__ typename A::Frag vfrag(int nt) const {
    if constexpr (DT == HCLSM_F32) {
      return caf4{__uint_as_float(v[0][nt]), __uint_as_float(v[1][nt]), __uint_as_float(v[2][nt]), __uint_as_float(v[3][nt])};
    } else {
      uint4 w;
      uint32_t* o = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
      for (int i = 0; i < 4; ++i) {       // halves nt & 1 of two keys' words side by side
        const uint32_t sel = (nt & 1) ? 0x07060302u : 0x05040100u;
        o[i] = __builtin_amdgcn_perm(v[2 * i + 1][nt >> 1], v[2 * i][nt >> 1], sel);
      }
      return ca_frag<DT>(w);
    }
  }
};

// Result of a row: in group K the lane holds columns c0 + 4 W g + W r + nt of tile nt, element r.
template <int DT, int DH, int K>
__device__ __forceinline__ void ca_few_store(const CaArgs& a, int64_t ob, const caf4* o, float f, bool in, int g) {
  using Gr = CaGroups<DT, DH>;
  if constexpr (K < Gr::N) {
    constexpr int F = Gr::first(K), W = Gr::width(K);
    const int col = 16 * F + 4 * W * g;
#pragma unroll
    for (int j = 0; j < W; ++j) {       // four columns at a time: elements 4j .. 4j + 3 of (r, nt) in order
      caf4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = in ? o[F + (4 * j + e) % W][(4 * j + e) / W] * f : 0.f;
      if (col + 4 * j < a.dh) {
        if (a.nsplit > 1) *reinterpret_cast<caf4*>(a.part + ob + col + 4 * j) = v;
        else ca_store4<DT>(a.o, ob + col + 4 * j, v);
      }
    }
    ca_few_store<DT, DH, K + 1>(a, ob, o, f, in, g);
  }
}

// NW waves share 16 QT rows and take every NW-th step of the keys, each with its own running maximum and sum; the waves'
// results are joined in LDS in a fixed order.  Keys and values go from global memory straight to the matrix unit's operand
// registers, one step ahead: no value is read by two waves, so LDS would only add a copy.
template <int DT, int DH, int NW, int QT>
__global__ void __launch_bounds__(64 * NW) ca_few_kernel(const CaArgs a) {
  using A = CaT<DT>;
  using Frag = typename A::Frag;
  using Step = CaStep<DT, DH>;
  constexpr int NC = DH / A::KS, ND = DH / 16, NPT = A::NPT, ESZ = (int)sizeof(typename A::T), SK = Step::SK;
  __shared__ float s_m[NW][QT][16], s_l[NW][QT][16];
  __shared__ caf4 s_o[NW > 1 ? NW / 2 : 1][QT][ND][64];

  CaWork w;
  if (!ca_work(a, w)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, g = lane >> 4;
  const int row0 = w.tile * 16 * QT;
  int k0, k1;
  ca_range(w.keys, a.nsplit, w.split, SK * NW, k0, k1);
  if (row0 >= w.rows) k1 = k0;
  const char* kp = a.k + (w.b * a.ksb + w.hk * a.ksh) * ESZ;
  const char* vp = a.v + (w.b * a.vsb + w.hk * a.vsh) * ESZ;
  const uint8_t* pad = a.pad ? a.pad + w.b * a.psb : nullptr;

  const int t0 = k0 + wave * SK;
  Step st;
  uint8_t flag = 0;
  auto get = [&](int t, Step& d) {
    d.load(a, kp, vp, t, k1 - 1, li, g);
    flag = pad != nullptr && lane < SK && t + lane < k1 ? pad[t + lane] : (uint8_t)0;
  };
  if (t0 < k1) get(t0, st);

  Frag q[QT][NC];
  {
    const char* qp = a.q + (w.b * a.qsb + (int64_t)w.hk * a.G * a.qsh) * ESZ;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const int r = row0 + 16 * t + li;
      int qi, hg;
      ca_row(a, r < w.rows ? r : 0, qi, hg);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int e = (4 * c + g) * A::EPC;
        uint4 f = {0, 0, 0, 0};
        if (r < w.rows && e < a.dh) f = *reinterpret_cast<const uint4*>(qp + (qi * a.qsl + hg * a.qsh + e) * ESZ);
        q[t][c] = ca_frag<DT>(f);
      }
    }
  }
  caf4 o[QT][ND];
  float m[QT], l[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    m[t] = -INFINITY;
    l[t] = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d) o[t][d] = caf4{0.f, 0.f, 0.f, 0.f};
  }

  for (int t = t0; t < k1; t += SK * NW) {
    const uint32_t live = (uint32_t)__ballot(lane < SK && t + lane < k1 && flag == 0);
    const bool full = live == (SK == 32 ? 0xffffffffu : 0xffffu);
    Step cur = st;
    if (t + SK * NW < k1) get(t + SK * NW, st);
    if (!full) {          // values of dead keys are zeros, whatever they held
#pragma unroll
      for (int p = 0; p < NPT; ++p)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (!(live >> (16 * p + 4 * g + r) & 1)) {
#pragma unroll
            for (int i = 0; i < Step::VW; ++i) cur.v[4 * p + r][i] = 0;
          }
    }
    caf4 s[QT][NPT];
#pragma unroll
    for (int p = 0; p < NPT; ++p) {
#pragma unroll
      for (int u = 0; u < QT; ++u) s[u][p] = caf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int u = 0; u < QT; ++u) s[u][p] = A::mma(ca_frag<DT>(cur.k[p][c]), q[u][c], s[u][p]);
    }
    Frag pf[QT];
#pragma unroll
    for (int u = 0; u < QT; ++u) {
      float mx = m[u];
#pragma unroll
      for (int p = 0; p < NPT; ++p)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (!full) s[u][p][r] = live >> (16 * p + 4 * g + r) & 1 ? s[u][p][r] : -INFINITY;
          mx = fmaxf(mx, s[u][p][r]);
        }
      mx = rows4_max(mx);
      const float base = mx == -INFINITY ? 0.f : mx * a.scale_log2;
      const float alpha = fast_exp2(m[u] * a.scale_log2 - base);
      const bool grew = mx > m[u];
      m[u] = mx;
      float sum = 0.f;
#pragma unroll
      for (int p = 0; p < NPT; ++p)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[u][p][r] = fast_exp2(s[u][p][r] * a.scale_log2 - base);
          sum += s[u][p][r];
        }
      l[u] = l[u] * alpha + sum;
      pf[u] = ca_pack<DT>(s[u]);
      if (__any(grew)) {
#pragma unroll
        for (int d = 0; d < ND; ++d) o[u][d] *= alpha;
      }
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const Frag f = cur.vfrag(d);
#pragma unroll
      for (int u = 0; u < QT; ++u) o[u][d] = A::mma(f, pf[u], o[u][d]);
    }
  }

  // join the waves: every wave scales to the common maximum, then halves add up in order
#pragma unroll
  for (int u = 0; u < QT; ++u) l[u] = rows4_sum(l[u]);
  float top[QT], sum[QT];
  if constexpr (NW > 1) {
    if (g == 0) {
#pragma unroll
      for (int u = 0; u < QT; ++u) { s_m[wave][u][li] = m[u]; s_l[wave][u][li] = l[u]; }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < QT; ++u) {
      top[u] = s_m[0][u][li];
#pragma unroll
      for (int i = 1; i < NW; ++i) top[u] = fmaxf(top[u], s_m[i][u][li]);
      const float base = top[u] == -INFINITY ? 0.f : top[u] * a.scale_log2;
      sum[u] = 0.f;
#pragma unroll
      for (int i = 0; i < NW; ++i) sum[u] += s_l[i][u][li] * fast_exp2(s_m[i][u][li] * a.scale_log2 - base);
      const float f = fast_exp2(m[u] * a.scale_log2 - base);
#pragma unroll
      for (int d = 0; d < ND; ++d) o[u][d] *= f;
    }
#pragma unroll
    for (int h = NW / 2; h >= 1; h >>= 1) {
      if (wave >= h && wave < 2 * h) {
#pragma unroll
        for (int u = 0; u < QT; ++u)
#pragma unroll
          for (int d = 0; d < ND; ++d) s_o[wave - h][u][d][lane] = o[u][d];
      }
      __syncthreads();
      if (wave < h) {
#pragma unroll
        for (int u = 0; u < QT; ++u)
#pragma unroll
          for (int d = 0; d < ND; ++d) o[u][d] += s_o[wave][u][d][lane];
      }
      __syncthreads();
    }
    if (wave != 0) return;
  } else {
#pragma unroll
    for (int u = 0; u < QT; ++u) { top[u] = m[u]; sum[u] = l[u]; }
  }

  const int all = a.Lq * a.G;
#pragma unroll
  for (int u = 0; u < QT; ++u) {
    const float inv = sum[u] > 0.f || sum[u] != sum[u] ? 1.f / sum[u] : 0.f;
    const int r = row0 + 16 * u + li;
    if (r >= all) continue;
    const bool in = r < w.rows;
    int qi, hg;
    ca_row(a, r, qi, hg);
    const int h = w.hk * a.G + hg;
    const float ls2 = in && sum[u] > 0.f ? top[u] * a.scale_log2 + __log2f(sum[u]) : in && sum[u] != sum[u] ? sum[u] : -INFINITY;
    const int64_t pr = ((int64_t)w.split * a.units + w.unit) * all + r;
    const int64_t ob = a.nsplit > 1 ? pr * a.dh : ((w.b * a.Lq + qi) * a.Hk * a.G + h) * (int64_t)a.dh;
    if (g == 0) {
      if (a.nsplit > 1) a.part_lse[pr] = ls2;
      else if (a.lse) a.lse[(w.b * a.Hk * a.G + h) * a.Lq + qi] = ls2 * HCLSM_LN2;
    }
    ca_few_store<DT, DH, 0>(a, ob, o[u], in ? inv : 0.f, in, g);
  }
}

}  // namespace hclsm
