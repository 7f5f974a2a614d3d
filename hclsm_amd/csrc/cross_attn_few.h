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

// One step's operands of a wave: SK = 16 NPT keys.
template <int DT, int DH> struct CaStep {
  using A = CaT<DT>;
  static constexpr int NPT = A::NPT, NC = DH / A::KS, ESZ = (int)sizeof(typename A::T), SK = 16 * NPT;
  static constexpr int VW = DH / 16 * ESZ / 4;      // words of a key's columns per lane
  uint4 k[NPT][NC];
  uint32_t v[NPT * 4][VW];

  static constexpr uint32_t NONE = 0xffffffffu;
  uint32_t koff, voff;       // bytes from a step's first key: row li at operand g; row 4g at this lane's columns

  __device__ __forceinline__ void init(const CaArgs& a, int li, int g) {
    koff = (uint32_t)li * (uint32_t)(a.ksl * ESZ) + 16 * g;
    voff = (uint32_t)(4 * g) * (uint32_t)(a.vsl * ESZ);
  }
  // keys kp / vp point at, n of them (past them, and past dh, loads are out of the buffer's range and give zeros)
  __device__ __forceinline__ void load(const CaArgs& a, const char* kp, const char* vp, int n, int li, int g) {
    const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc((void*)kp, 0, 0x7fffffff, kRawBufferWord3);
    const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc((void*)vp, 0, 0x7fffffff, kRawBufferWord3);
#pragma unroll
    for (int t = 0; t < NPT; ++t) {
      const uint32_t row = 16 * t + li < n ? koff : NONE;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const uint32_t o = (4 * c + g) * A::EPC < a.dh ? row : NONE;
        k[t][c] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(
            rk, (int)(o == NONE ? o : o + 64 * c), t * 16 * (int)(a.ksl * ESZ), 0));
      }
    }
#pragma unroll
    for (int t = 0; t < NPT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        load_v<0>(a, rv, 16 * t + 4 * g + r < n ? voff : NONE, (16 * t + r) * (int)(a.vsl * ESZ), li, v[4 * t + r]);
  }
  template <int K>
  __device__ __forceinline__ void load_v(const CaArgs& a, __amdgpu_buffer_rsrc_t rv, uint32_t off, int so, int li, uint32_t* w) {
    if constexpr (K < CaGroups<DT, DH>::N) {
      constexpr int F = CaGroups<DT, DH>::first(K), W = CaGroups<DT, DH>::width(K), WORDS = W * ESZ / 4;
      const int col = 16 * F + W * li;
      const int o = (int)(off != NONE && col < a.dh ? off + col * ESZ : NONE);
      uint32_t* d = w + F * ESZ / 4;
      if constexpr (WORDS == 4) {
        const uint4 x = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rv, o, so, 0));
        d[0] = x.x; d[1] = x.y; d[2] = x.z; d[3] = x.w;
      } else if constexpr (WORDS == 2) {
        const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(rv, o, so, 0));
        d[0] = x.x; d[1] = x.y;
      } else {
        d[0] = __builtin_amdgcn_raw_buffer_load_b32(rv, o, so, 0);
      }
      load_v<K + 1>(a, rv, off, so, li, w);
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
        else ca_store_out<DT>(a, ob + col + 4 * j, v);
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
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, g = lane >> 4;
  const int row0 = w.tile * 16 * QT;
  int k0, k1;
  ca_range(w.keys, a.nsplit, w.split, SK * NW, k0, k1);
  if (row0 >= w.rows) k1 = k0;
  const char* kp = a.k + (w.b * a.ksb + w.hk * a.ksh) * ESZ;
  const char* vp = a.v + (w.b * a.vsb + w.hk * a.vsh) * ESZ;
  const uint8_t* pad = a.pad ? a.pad + w.b * a.psb : nullptr;

  const int t0 = k0 + wave * SK;
  Step st;
  st.init(a, li, g);
  uint8_t flag = 0;
  auto get = [&](int t, Step& d) {
    d.load(a, kp + t * a.ksl * ESZ, vp + t * a.vsl * ESZ, k1 - t, li, g);
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
    m[t] = CA_LOW;
    l[t] = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d) o[t][d] = caf4{0.f, 0.f, 0.f, 0.f};
  }

  for (int t = t0; t < k1; t += SK * NW) {
    const uint32_t live = (uint32_t)__ballot(lane < SK && t + lane < k1 && flag == 0);
    const bool full = live == (SK == 32 ? 0xffffffffu : 0xffffu);
    Step cur = st;
    if (t + SK * NW < k1) get(t + SK * NW, st);
    if (pad != nullptr && !full) {          // values of masked keys are zeros, whatever they held
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
    float top[QT];
    bool grew = false;
#pragma unroll
    for (int u = 0; u < QT; ++u) {
      if (!full) {
#pragma unroll
        for (int p = 0; p < NPT; ++p)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[u][p][r] = live >> (16 * p + 4 * g + r) & 1 ? s[u][p][r] : -INFINITY;
      }
      float mx = s[u][0][0];
#pragma unroll
      for (int p = 0; p < NPT; ++p)
#pragma unroll
        for (int r = 0; r < 4; r += 2) mx = ca_max3(mx, s[u][p][r], s[u][p][r + 1]);
      top[u] = ca_rows4_max(mx) * a.scale_log2;
      grew |= !(top[u] <= m[u] + CA_SLACK);
    }
    if (__any(grew)) {         // as in ca_fwd_kernel
#pragma unroll
      for (int u = 0; u < QT; ++u) {
        const float to = top[u] <= m[u] + CA_SLACK ? m[u] : top[u];
        const float alpha = fast_exp2(m[u] - to);
        m[u] = to;
        l[u] *= alpha;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[u][d] *= alpha;
      }
    }
    Frag pf[QT];
#pragma unroll
    for (int u = 0; u < QT; ++u) {
#pragma unroll
      for (int p = 0; p < NPT; ++p)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[u][p][r] = fast_exp2(s[u][p][r] * a.scale_log2 - m[u]);
          l[u] += s[u][p][r];
        }
      pf[u] = ca_pack<DT>(s[u]);
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
      for (int i = 1; i < NW; ++i) top[u] = __builtin_elementwise_maximum(top[u], s_m[i][u][li]);
      sum[u] = 0.f;
#pragma unroll
      for (int i = 0; i < NW; ++i) sum[u] += s_l[i][u][li] * fast_exp2(s_m[i][u][li] - top[u]);
      const float f = fast_exp2(m[u] - top[u]);
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
    const float ls2 = in && sum[u] > 0.f ? top[u] + __log2f(sum[u]) : in && sum[u] != sum[u] ? sum[u] : -INFINITY;
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
