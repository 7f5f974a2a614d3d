// Cross attention of few rows of a unit (one query and its shared heads, or a frame's slots), where reading the keys and
// values is the work: at most 16 rows, or 32 of short heads and in the backward (ca_forward_plan, ca_backward_plan).
#pragma once

#include "cross_attn_stage.h"

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
  static __device__ __forceinline__ void load_v(const CaArgs& a, __amdgpu_buffer_rsrc_t rv, uint32_t off, int so, int li, uint32_t* w) {
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
  __device__ __forceinline__ typename A::Frag vfrag(int nt) const { return column(v, nt); }
  static __device__ __forceinline__ typename A::Frag column(const uint32_t (*v)[VW], int nt) {
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

// Result of a row: in group K the lane holds columns c0 + 4 W g + W r + nt of tile nt, element r.  put(column, four values).
template <int DT, int DH, int K = 0, typename F>
__device__ __forceinline__ void ca_few_store(int dh, const caf4* o, float f, bool in, int g, F put) {
  using Gr = CaGroups<DT, DH>;
  if constexpr (K < Gr::N) {
    constexpr int F0 = Gr::first(K), W = Gr::width(K);
    const int col = 16 * F0 + 4 * W * g;
#pragma unroll
    for (int j = 0; j < W; ++j) {       // four columns at a time: elements 4j .. 4j + 3 of (r, nt) in order
      caf4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = in ? o[F0 + (4 * j + e) % W][(4 * j + e) / W] * f : 0.f;
      if (col + 4 * j < dh) put(col + 4 * j, v);
    }
    ca_few_store<DT, DH, K + 1>(dh, o, f, in, g, put);
  }
}

// NW waves share 16 QT rows and take every NW-th step of the keys, each with its own running maximum and sum; the waves'
// results are joined in LDS in a fixed order.  Keys and values go from global memory straight to the matrix unit's operand
// registers, one step ahead: no value is read by two waves, so LDS would only add a copy.
// What bounds it: reading k and v.  Measured (bf16): one query on 100352 keys, 16 heads of 128 on 4, keys split over 64
// workgroups per key head: 41 us, 4.9 TB/s, and 5 us to join; 64 single queries on up to 1568 keys, 12 heads of 64: 46 us,
// 4.2 TB/s; float32, 32 slots on 196 tokens of 64 frames, 6 heads of 64: 17 us, 2.6 TB/s (two steps of keys to a wave: its
// time is the wait for the first and the joining).  A 1 GiB copy reaches 5.1 TB/s.
template <int DT, int DH, int NW, int QT>
__global__ void __launch_bounds__(64 * NW) ca_few_kernel(const CaArgs a) {
  using A = CaT<DT>;
  using Frag = typename A::Frag;
  using Step = CaStep<DT, DH>;
  constexpr int NC = DH / A::KS, ND = DH / 16, NPT = A::NPT, ESZ = (int)sizeof(typename A::T), SK = Step::SK;
  constexpr int PARTS = DT == HCLSM_F32 ? 1 : 2;
  __shared__ float s_m[NW][QT][16], s_l[NW][QT][16];
  static_assert(NW >= 2 && (NW & (NW - 1)) == 0, "waves are joined by halves");
  __shared__ caf4 s_o[NW / 2][QT][ND][64];

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
      grew |= !(top[u] <= m[u] + CA_SLACK<DT>);
    }
    if (__any(grew)) {         // as in ca_fwd_kernel
#pragma unroll
      for (int u = 0; u < QT; ++u) {
        const float to = top[u] <= m[u] + CA_SLACK<DT> ? m[u] : top[u] - CA_BELOW<DT>;
        const float alpha = fast_exp2(m[u] - to);
        m[u] = to;
        l[u] *= alpha;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[u][d] *= alpha;
      }
    }
    Frag pf[QT][PARTS];
#pragma unroll
    for (int u = 0; u < QT; ++u) {
#pragma unroll
      for (int p = 0; p < NPT; ++p)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[u][p][r] = fast_exp2(s[u][p][r] * a.scale_log2 - m[u]);
          l[u] += s[u][p][r];
        }
      ca_pack_parts<DT, PARTS>(s[u], pf[u]);
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const Frag f = cur.vfrag(d);
#pragma unroll
      for (int u = 0; u < QT; ++u)
#pragma unroll
        for (int e = 0; e < PARTS; ++e) o[u][d] = A::mma(f, pf[u][e], o[u][d]);
    }
  }

  // join the waves: every wave scales to the common maximum, then halves add up in order
#pragma unroll
  for (int u = 0; u < QT; ++u) l[u] = rows4_sum(l[u]);
  float top[QT], sum[QT];
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
    ca_few_store<DT, DH>(a.dh, o[u], inv, in, g, [&](int col, caf4 v) {
      if (a.nsplit > 1) *reinterpret_cast<caf4*>(a.part + ob + col) = v;
      else ca_store_out<DT>(a, ob + col, v);
    });
  }
}

// Gradients of at most 32 rows of a unit in one pass over its keys: all rows are at hand, so a key's dk and dv are whole
// as soon as the key has been read, and only dq is summed over the keys (over the waves and, when the keys are
// split over workgroups, by ca_sum_kernel).  Both orientations of the scores are formed, S^T (a lane per row) for
// dQ^T = K^T ds^T and S (a lane per key) for dV^T = g^T p and dK^T = Q^T ds: the key's operand registers serve both, and
// moving ds between the lanes would cost more than the second product.  What bounds it: reading q, g, out and k, v once
// and writing dq, dk, dv.  Measured: 32 slots on 196 tokens of 256 frames, 6 heads of 64, bf16: 54 us, 3.4 TB/s (the two
// tiled kernels: 67 us); matrix unit busy 10% of the cycles, vector unit 32%: a wave has one or two steps of keys and waits
// for the rows, and for each step's keys, with nothing else to do.
// Two workgroups to a CU are asked for with heads up to 64: float16 would take one register more than that leaves.
template <int DT, int DH, int NW>
__global__ void __launch_bounds__(64 * NW, DH <= 64 ? 2 : 1) ca_few_bwd_kernel(const CaArgs a) {
  using A = CaT<DT>;
  using Frag = typename A::Frag;
  using Tile = CaTile<DT, DH>;
  using Step = CaStep<DT, DH>;
  constexpr int NT = 64 * NW, QT = 2, R = 16 * QT, NC = DH / A::KS, ND = DH / 16, NPT = A::NPT, SK = Step::SK;
  constexpr int ESZ = (int)sizeof(typename A::T), VW = Step::VW, RU = QT / NPT;
  constexpr int PARTS = DT == HCLSM_F32 ? 1 : 2;
  using Stage = CaStage<DT, DH, NT, R>;
  __shared__ __attribute__((aligned(16))) char tq[Stage::BYTES];
  __shared__ __attribute__((aligned(16))) char tg[Stage::BYTES];
  __shared__ __attribute__((aligned(16))) float stat[2 * R];       // log-sums (log2), negated deltas
  __shared__ caf4 s_dq[NW / 2][QT][ND][64];

  CaWork w;
  if (!ca_work(a, w)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, g = lane >> 4;
  int k0, k1;
  ca_range(a.Lk, a.nsplit, w.split, SK * NW, k0, k1);        // every key: dk and dv are written for all of them
  const char* kp = a.k + (w.b * a.ksb + w.hk * a.ksh) * ESZ;
  const char* vp = a.v + (w.b * a.vsb + w.hk * a.vsh) * ESZ;
  const uint8_t* pad = a.pad ? a.pad + w.b * a.psb : nullptr;
  const int h0 = w.hk * a.G;

  const uint32_t koff = (uint32_t)li * (uint32_t)(a.ksl * ESZ) + 16 * g, voff = (uint32_t)li * (uint32_t)(a.vsl * ESZ) + 16 * g;
  const uint32_t coff = (uint32_t)(4 * g) * (uint32_t)(a.ksl * ESZ);
  constexpr uint32_t NONE = 0xffffffffu;
  uint4 k[NPT][NC], v[NPT][NC];       // a step's keys and values along their rows, and the keys by column
  uint32_t kc[NPT * 4][VW];
  uint8_t flag = 0;
  auto load = [&](int t0) __attribute__((always_inline)) {
    const int n = w.keys - t0;
    flag = pad != nullptr && lane < SK && lane < n ? pad[t0 + lane] : (uint8_t)0;
    const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc((void*)(kp + t0 * a.ksl * ESZ), 0, 0x7fffffff, kRawBufferWord3);
    const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc((void*)(vp + t0 * a.vsl * ESZ), 0, 0x7fffffff, kRawBufferWord3);
#pragma unroll
    for (int p = 0; p < NPT; ++p) {
      const bool in = 16 * p + li < n;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const bool have = in && (4 * c + g) * A::EPC < a.dh;
        k[p][c] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(
            rk, (int)(have ? koff + 64 * c : NONE), 16 * p * (int)(a.ksl * ESZ), 0));
        v[p][c] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(
            rv, (int)(have ? voff + 64 * c : NONE), 16 * p * (int)(a.vsl * ESZ), 0));
      }
    }
#pragma unroll
    for (int p = 0; p < NPT; ++p)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        Step::template load_v<0>(a, rk, 16 * p + 4 * g + r < n ? coff : NONE, (16 * p + r) * (int)(a.ksl * ESZ), li, kc[4 * p + r]);
  };

  Stage sq, sg;
  sq.init_rows(a, a.qsl, a.qsh, 0, R);
  sg.init_rows(a, a.gsl, a.gsh, 0, R);
  sq.load(a.q + (w.b * a.qsb + h0 * a.qsh) * ESZ, w.rows, tq, wave);
  sg.load(a.g + (w.b * a.gsb + h0 * a.gsh) * ESZ, w.rows, tg, wave);
  if (k0 + wave * SK < k1) load(k0 + wave * SK);      // on their way while the rows are prepared
  ca_wait_vmem();
  __syncthreads();
  Frag q[QT][NC], go[QT][NC];
#pragma unroll
  for (int t = 0; t < QT; ++t)
#pragma unroll
    for (int c = 0; c < NC; ++c) { q[t][c] = Tile::frag(tq, 16 * t, c, li, g); go[t][c] = Tile::frag(tg, 16 * t, c, li, g); }
  static_assert(NW >= QT, "a wave per tile of rows");
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    if (wave != t) continue;
    const int r = 16 * t + li;
    const bool in = r < w.rows;
    int qi, hg;
    ca_row(a, in ? r : 0, qi, hg);
    const int64_t ob = ((w.b * a.Lq + qi) * a.Hk * a.G + h0 + hg) * (int64_t)a.dh * ESZ;
    uint4 fo[NC], fl[NC];
    ca_row_frags<DT, DH>(a.o + ob, g, a.dh, in, fo);
    ca_row_frags<DT, DH>(a.olo + ob, g, a.dh, in && a.olo != nullptr, fl);
    float d = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      d = ca_dot<DT>(__builtin_bit_cast(uint4, go[t][c]), fo[c], d);
      d = ca_dot<DT>(__builtin_bit_cast(uint4, go[t][c]), fl[c], d);
    }
    d = rows4_sum(d);
    const float ls = in ? a.lse[(w.b * a.Hk * a.G + h0 + hg) * a.Lq + qi] : -INFINITY;
    if (g == 0) {
      stat[r] = ls == -INFINITY ? INFINITY : ls * HCLSM_LOG2E;
      stat[R + r] = -d;
    }
  }
  __syncthreads();
  float lse2[QT];
  caf4 nd[QT], lsr[QT], ndr[QT];        // of row li; of rows 4g .. 4g + 3
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    lse2[t] = stat[16 * t + li];
    const float d = stat[R + 16 * t + li];
    nd[t] = caf4{d, d, d, d};
    lsr[t] = *reinterpret_cast<const caf4*>(stat + 16 * t + 4 * g) - CA_P_SHIFT<DT>;
    ndr[t] = *reinterpret_cast<const caf4*>(stat + R + 16 * t + 4 * g);
  }

  caf4 dq[QT][ND];
  float up[QT];         // float16: factor of the row's ds in this wave
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    up[t] = ca_pow2(CA_F16_START);
#pragma unroll
    for (int d = 0; d < ND; ++d) dq[t][d] = caf4{0.f, 0.f, 0.f, 0.f};
  }

  for (int t0 = k0 + wave * SK; t0 < k1; t0 += SK * NW) {
    const int n = w.keys - t0;                                      // keys there are from t0 on
    const uint32_t live = (uint32_t)__ballot(lane < SK && lane < n && flag == 0);
    const bool full = live == (SK == 32 ? 0xffffffffu : 0xffffu);
    if (pad != nullptr && !full) {
#pragma unroll
      for (int p = 0; p < NPT; ++p)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (!(live >> (16 * p + 4 * g + r) & 1)) {
#pragma unroll
            for (int i = 0; i < VW; ++i) kc[4 * p + r][i] = 0;
          }
    }

    // dq: a lane per row
    if (a.dq != nullptr) {
      caf4 s[QT][NPT], dp[QT][NPT];
#pragma unroll
      for (int p = 0; p < NPT; ++p) {
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          s[t][p] = caf4{0.f, 0.f, 0.f, 0.f};
          dp[t][p] = nd[t];
        }
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int t = 0; t < QT; ++t) {
            s[t][p] = A::mma(ca_frag<DT>(k[p][c]), q[t][c], s[t][p]);
            dp[t][p] = A::mma(ca_frag<DT>(v[p][c]), go[t][c], dp[t][p]);
          }
      }
      Frag ds[QT][PARTS];
#pragma unroll
      for (int t = 0; t < QT; ++t) {
#pragma unroll
        for (int p = 0; p < NPT; ++p)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            dp[t][p][r] *= fast_exp2(s[t][p][r] * a.scale_log2 - lse2[t]);
            if (!full) dp[t][p][r] = live >> (16 * p + 4 * g + r) & 1 ? dp[t][p][r] : 0.f;
          }
        if constexpr (CA_RANGED<DT>) {
          const float most = ca_scale_most<NPT>(dp[t], up[t]);
          if (__any(most > CA_F16_MOST)) {
            const float f = ca_lowered(ca_rows4_max(most));
            up[t] *= f;
#pragma unroll
            for (int p = 0; p < NPT; ++p) dp[t][p] *= f;
#pragma unroll
            for (int d = 0; d < ND; ++d) dq[t][d] *= f;
          }
        }
        ca_pack_parts<DT, PARTS>(dp[t], ds[t]);
      }
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const Frag f = Step::column(kc, d);
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
          for (int e = 0; e < PARTS; ++e) dq[t][d] = A::mma(f, ds[t][e], dq[t][d]);
      }
    }
    // dk, dv: a lane per key; a key that is not live spoils no column but its own, which is written as zeros
    Frag p2[NPT][RU][PARTS], ds2[NPT][RU][PARTS];
    float down[NPT];      // float16: 1 / factor of the key's ds
#pragma unroll
    for (int p = 0; p < NPT; ++p) {
      caf4 s[QT], dp[QT];
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        s[t] = caf4{0.f, 0.f, 0.f, 0.f};
        dp[t] = ndr[t];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          s[t] = A::mma(q[t][c], ca_frag<DT>(k[p][c]), s[t]);
          dp[t] = A::mma(go[t][c], ca_frag<DT>(v[p][c]), dp[t]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[t][r] = fast_exp2(s[t][r] * a.scale_log2 - lsr[t][r]);
          dp[t][r] *= s[t][r];
        }
      }
      if constexpr (CA_RANGED<DT>) {
        const float f = ca_fitted(ca_rows4_max(ca_scale_most<QT>(dp, 1.f)));
        down[p] = ca_unscaled(f) * CA_P_DOWN<DT>;
#pragma unroll
        for (int t = 0; t < QT; ++t) dp[t] *= f;
      }
#pragma unroll
      for (int u = 0; u < RU; ++u) {
        ca_pack_parts<DT, PARTS>(&s[u * NPT], p2[p][u]);
        ca_pack_parts<DT, PARTS>(&dp[u * NPT], ds2[p][u]);
      }
    }
    if (t0 + SK * NW < k1) load(t0 + SK * NW);
    if (a.dk == nullptr) continue;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      caf4 dk[NPT], dv[NPT];
#pragma unroll
      for (int p = 0; p < NPT; ++p) dk[p] = dv[p] = caf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < RU; ++u) {
        const Frag fg = Tile::frag_t(tg, 16 * NPT * u, d, li, g);
        const Frag fq = Tile::frag_t(tq, 16 * NPT * u, d, li, g);
#pragma unroll
        for (int p = 0; p < NPT; ++p)
#pragma unroll
          for (int e = 0; e < PARTS; ++e) {
            dv[p] = A::mma(fg, p2[p][u][e], dv[p]);
            dk[p] = A::mma(fq, ds2[p][u][e], dk[p]);
          }
      }
#pragma unroll
      for (int p = 0; p < NPT; ++p) {
        const int key = t0 + 16 * p + li;
        if (key < k1 && 16 * d + 4 * g < a.dh) {
          const bool in = live >> (16 * p + li) & 1;
          const caf4 zero = {0.f, 0.f, 0.f, 0.f};
          const int64_t i = ((w.b * a.Lk + key) * a.Hk + w.hk) * (int64_t)a.dh + 16 * d + 4 * g;
          if constexpr (CA_RANGED<DT>) {
            dk[p] *= down[p];
            dv[p] *= CA_P_DOWN<DT>;
          }
          ca_store4<DT>(a.dk, i, in ? dk[p] * a.scale : zero);
          ca_store4<DT>(a.dv, i, in ? dv[p] : zero);
        }
      }
    }
  }
  if (a.dq == nullptr) return;

  // dq of the waves, added in a fixed order
  if constexpr (CA_RANGED<DT>) {
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
      for (int d = 0; d < ND; ++d) dq[t][d] *= ca_unscaled(up[t]);
  }
#pragma unroll
  for (int h = NW / 2; h >= 1; h >>= 1) {
    if (wave >= h && wave < 2 * h) {
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int d = 0; d < ND; ++d) s_dq[wave - h][t][d][lane] = dq[t][d];
    }
    __syncthreads();
    if (wave < h) {
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int d = 0; d < ND; ++d) dq[t][d] += s_dq[wave][t][d][lane];
    }
    __syncthreads();
  }
  if (wave != 0) return;
  const int all = a.Lq * a.G;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = 16 * t + li;
    if (r >= all) continue;
    int qi, hg;
    ca_row(a, r, qi, hg);
    const int64_t ob = a.nsplit > 1 ? (((int64_t)w.split * a.units + w.unit) * all + r) * a.dh
                                    : ((w.b * a.Lq + qi) * a.Hk * a.G + h0 + hg) * (int64_t)a.dh;
    ca_few_store<DT, DH>(a.dh, dq[t], a.scale, r < w.rows, g, [&](int col, caf4 x) {
      if (a.nsplit > 1) *reinterpret_cast<caf4*>(a.part + ob + col) = x;
      else ca_store4<DT>(a.dq, ob + col, x);
    });
  }
}

}  // namespace hclsm
