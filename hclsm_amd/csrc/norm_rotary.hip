// Norms of queries and keys for each head and their position rotation, forward and backward (gfx950).
//
// One row is one head of one token: dh elements x.  With r = rsqrt(mean(x^2) + eps) (1 without the norm) and the
// weight w (1 without one),
//     n = x r,   y = R(n w),
// where R turns pair i (elements (i, i + rot/2) or (2i, 2i + 1) of the first rot) by position * frequency_i and
// scales it by an amplitude; elements from rot on pass through.  R^T, which turns back, gives the gradients:
//     d = R^T g,   dw = sum over rows of d n,   dx = r (d w - n mean(d w n)).
// Everything between the load and the one rounding at the store is float32.  The angle is formed in turns,
// t = position * (frequency / 2 pi), in float64, and only t - rint(t) is rounded to float32: a position of 2^31
// still leaves 2^-22 turns.
//
// What bounds it: HBM (2 bytes in, 2 out per bf16 element against about 10 float operations).  A row is spread over
// G lanes that hold V pairs each (two vectors of V elements per lane and row: 16 B loads when rot, dh, the strides
// and the addresses allow it, else 8, 4 or 2 B); one lane group takes up to HPL heads of a token, so an angle (about
// 60 instructions, part of them float64) is shared by HPL rows and HPL rows' loads are in flight together.
#include "internal.h"

namespace hclsm {

constexpr int NR_THREADS = 256;
constexpr int NR_HPL = 4;             // heads of a token per lane group
constexpr int NR_MAX_DH = 256;
constexpr int NR_BWD_BLOCKS = 1024;   // most workgroups (= partial sums of dw) per tensor of the backward
constexpr int NR_FWD_BLOCKS = 1 << 20;   // of the forward: a launch has fewer than 2^32 threads, the rest is looped over

// One tensor of heads as the kernels read it.
struct NrTensor {
  const char *x, *g;            // input; gradient of the output (backward)
  char* y;                      // output, or gradient of the input: contiguous [B, L, H, dh]
  const void* w;                // [dh] or null
  const void* pos;              // null: the token's index
  float* part;                  // backward: [blocks][dh] partial sums of dw, null when not wanted
  int64_t xsb, xsl, xsh, gsb, gsl, gsh;   // element strides
  int64_t psb, psl;
  int pos_dtype, w_dtype;
  uint32_t L, H, chunks;        // chunks = ceil(H / HPL)
  uint32_t items;               // B * L * chunks
  uint32_t blocks;
};

struct NrArgs {
  NrTensor t[2];
  const double* turns;          // [rot / 2]: frequency / 2 pi
  int dh, rot;
  float amp, eps;
};

// V elements of 2 or 4 bytes as one access
template <int BYTES> struct NrWord;
template <> struct NrWord<16> { using T = uint4; };
template <> struct NrWord<8> { using T = uint2; };
template <> struct NrWord<4> { using T = uint32_t; };
template <> struct NrWord<2> { using T = uint16_t; };

template <int DT, int V> struct NrVec {
  using E = typename Elem<DT>::T;
  using W = typename NrWord<V * (int)sizeof(E)>::T;
  E e[V];
  __device__ __forceinline__ void load(const E* p) {
    *this = __builtin_bit_cast(NrVec, *reinterpret_cast<const W*>(p));
  }
  __device__ __forceinline__ void store(E* p) const {
    *reinterpret_cast<W*>(p) = __builtin_bit_cast(W, *this);
  }
  __device__ __forceinline__ float get(int i) const { return Elem<DT>::ld(&e[i]); }
  __device__ __forceinline__ void set(int i, float v) { Elem<DT>::st(&e[i], v); }
};

__device__ __forceinline__ float nr_weight(const void* w, int dt, int i) {
  if (w == nullptr) return 1.f;
  if (dt == HCLSM_F32) return reinterpret_cast<const float*>(w)[i];
  if (dt == HCLSM_BF16) return bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(w)[i]);
  return (float)reinterpret_cast<const _Float16*>(w)[i];
}

// Sum over the G lanes of a group (G a power of two, groups aligned), the same bits in every lane.
__device__ __forceinline__ float nr_group_sum(float v, int G) {
  for (int o = 1; o < G; o <<= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// V: pairs per lane and unit.  NU: units per lane.  A unit is two vectors of V elements: unit u < rot / 2V holds pairs
// uV .. uV + V - 1 (INTER: elements 2uV .. 2uV + 2V - 1, else uV .. and rot/2 + uV ..), later units hold
// the elements that pass through, 2V each, the last one possibly V.
template <int DT, int V, int NU, bool INTER, bool NORM, bool BWD>
__global__ void __launch_bounds__(NR_THREADS) norm_rotary_kernel(NrArgs a, int G) {
  using E = typename Elem<DT>::T;
  using Vec = NrVec<DT, V>;
  const bool second = blockIdx.x >= a.t[0].blocks;
  const NrTensor& t = a.t[second ? 1 : 0];
  const uint32_t blk = second ? blockIdx.x - a.t[0].blocks : blockIdx.x;
  const int groups = NR_THREADS / G;
  const int grp = threadIdx.x / G, gl = threadIdx.x & (G - 1);
  const int half = a.rot >> 1, npair = half / V;

  // this lane's elements: column of each unit's two vectors, -1 where there is none
  int col[NU][2];
  bool pair[NU];
  float w[NU][2 * V];
#pragma unroll
  for (int k = 0; k < NU; ++k) {
    const int u = gl + k * G;
    pair[k] = u < npair;
    col[k][0] = pair[k] ? (INTER ? 2 * u * V : u * V) : a.rot + (u - npair) * 2 * V;
    col[k][1] = pair[k] && !INTER ? half + u * V : col[k][0] + V;
    if (col[k][0] >= a.dh) col[k][0] = -1;
    if (col[k][1] >= a.dh) col[k][1] = -1;
    if (NORM) {
#pragma unroll
      for (int j = 0; j < 2 * V; ++j) {
        const int c = col[k][j / V];
        w[k][j] = c < 0 ? 0.f : nr_weight(t.w, t.w_dtype, c + j % V);
      }
    }
  }
  float gw[NU][2 * V];
  if (BWD) {
#pragma unroll
    for (int k = 0; k < NU; ++k)
#pragma unroll
      for (int j = 0; j < 2 * V; ++j) gw[k][j] = 0.f;
  }

  // Lanes past the last item keep going with no head of their own (the sums below need whole groups).  The step
  // is 64 bits wide: item + stride may pass 2^32.
  const uint64_t step = (uint64_t)t.blocks * groups;
  for (uint64_t it = (uint64_t)blk * groups; it < t.items; it += step) {
    const uint32_t item = (uint32_t)(it + grp < t.items ? it + grp : t.items - 1);
    const bool live = it + grp < t.items;
    const uint32_t tok = item / t.chunks, c = item - tok * t.chunks;
    const uint32_t b = tok / t.L, l = tok - b * t.L;
    const uint32_t h0 = c * NR_HPL;
    const int nh = !live ? 0 : (int)(t.H - h0 < NR_HPL ? t.H - h0 : NR_HPL);

    // loads of every head first
    Vec x[NR_HPL][NU][2], g[BWD ? NR_HPL : 1][NU][2];
    const E* xp = reinterpret_cast<const E*>(t.x) + b * t.xsb + l * t.xsl + h0 * t.xsh;
    const E* gp = BWD ? reinterpret_cast<const E*>(t.g) + b * t.gsb + l * t.gsl + h0 * t.gsh : nullptr;
#pragma unroll
    for (int h = 0; h < NR_HPL; ++h) {
#pragma unroll
      for (int k = 0; k < NU; ++k)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          x[h][k][s] = Vec{};
          if (BWD) g[h][k][s] = Vec{};
          if (h < nh && col[k][s] >= 0) {
            x[h][k][s].load(xp + h * t.xsh + col[k][s]);
            if (BWD) g[h][k][s].load(gp + h * t.gsh + col[k][s]);
          }
        }
    }

    // cos and sin of this lane's pairs
    float cs[NU][V], sn[NU][V];
    int64_t p = l;
    if (t.pos) {
      const int64_t pi = b * t.psb + l * t.psl;
      p = t.pos_dtype == HCLSM_POS_I32 ? (int64_t)reinterpret_cast<const int32_t*>(t.pos)[pi]
                                       : reinterpret_cast<const int64_t*>(t.pos)[pi];
    }
#pragma unroll
    for (int k = 0; k < NU; ++k) {
      if (pair[k]) {
        const int u = gl + k * G;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          double tr = (double)p * a.turns[u * V + j];
          tr -= rint(tr);
          sincospif(2.f * (float)tr, &sn[k][j], &cs[k][j]);
          sn[k][j] *= a.amp;
          cs[k][j] *= a.amp;
        }
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) { cs[k][j] = 1.f; sn[k][j] = 0.f; }
      }
    }

    E* yp = reinterpret_cast<E*>(t.y) + ((int64_t)tok * t.H + h0) * a.dh;
#pragma unroll
    for (int h = 0; h < NR_HPL; ++h) {
      if (!NORM && h >= nh) continue;
      float r = 1.f;
      if (NORM) {
        float ss = 0.f;
#pragma unroll
        for (int k = 0; k < NU; ++k)
#pragma unroll
          for (int j = 0; j < 2 * V; ++j) { const float v = x[h][k][j / V].get(j % V); ss += v * v; }
        r = rsqrtf(nr_group_sum(ss, G) / (float)a.dh + a.eps);
      }
      if (!BWD) {
        if (h < nh) {
#pragma unroll
          for (int k = 0; k < NU; ++k) {
            float e[2 * V];
#pragma unroll
            for (int j = 0; j < 2 * V; ++j) {
              e[j] = x[h][k][j / V].get(j % V);
              if (NORM) e[j] = e[j] * r * w[k][j];
            }
            Vec o[2];
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const int ia = INTER ? 2 * j : j, ib = INTER ? 2 * j + 1 : V + j;
              const float ya = e[ia] * cs[k][j] - e[ib] * sn[k][j], yb = e[ib] * cs[k][j] + e[ia] * sn[k][j];
              o[ia / V].set(ia % V, pair[k] ? ya : e[ia]);
              o[ib / V].set(ib % V, pair[k] ? yb : e[ib]);
            }
#pragma unroll
            for (int s = 0; s < 2; ++s)
              if (col[k][s] >= 0) o[s].store(yp + h * a.dh + col[k][s]);
          }
        }
      } else {
        float d[NU][2 * V], dot = 0.f;
#pragma unroll
        for (int k = 0; k < NU; ++k) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const int ia = INTER ? 2 * j : j, ib = INTER ? 2 * j + 1 : V + j;
            const float ga = g[h][k][ia / V].get(ia % V), gb = g[h][k][ib / V].get(ib % V);
            d[k][ia] = pair[k] ? ga * cs[k][j] + gb * sn[k][j] : ga;
            d[k][ib] = pair[k] ? gb * cs[k][j] - ga * sn[k][j] : gb;
          }
#pragma unroll
          for (int j = 0; j < 2 * V; ++j) {
            const float n = x[h][k][j / V].get(j % V) * r;
            if (h < nh) gw[k][j] += d[k][j] * n;
            d[k][j] *= w[k][j];
            dot += d[k][j] * n;
          }
        }
        dot = nr_group_sum(dot, G) / (float)a.dh;
        if (h < nh) {
#pragma unroll
          for (int k = 0; k < NU; ++k) {
            Vec o[2];
#pragma unroll
            for (int j = 0; j < 2 * V; ++j)
              o[j / V].set(j % V, r * (d[k][j] - x[h][k][j / V].get(j % V) * r * dot));
#pragma unroll
            for (int s = 0; s < 2; ++s)
              if (col[k][s] >= 0) o[s].store(yp + h * a.dh + col[k][s]);
          }
        }
      }
    }
  }

  if (BWD) {
    // dw of this workgroup: the groups' sums added in the groups' order
    __shared__ float red[NR_THREADS * 2 * V * NU];
    if (t.part == nullptr) return;
    const int width = G * NU * 2 * V;
#pragma unroll
    for (int k = 0; k < NU; ++k)
#pragma unroll
      for (int j = 0; j < 2 * V; ++j) red[grp * width + (k * 2 * V + j) * G + gl] = gw[k][j];
    __syncthreads();
    if (grp == 0) {
#pragma unroll
      for (int k = 0; k < NU; ++k)
#pragma unroll
        for (int j = 0; j < 2 * V; ++j) {
          if (col[k][j / V] < 0) continue;
          float s = 0.f;
          for (int q = 0; q < groups; ++q) s += red[q * width + (k * 2 * V + j) * G + gl];
          t.part[(int64_t)blk * a.dh + col[k][j / V] + j % V] = s;
        }
    }
  }
}

// gw[c] = sum over blocks of part[block][c], in a fixed order: 16 columns x 16 row lanes per workgroup.
__global__ void __launch_bounds__(256) norm_rotary_dw_kernel(const float* p0, uint32_t n0, void* w0, int dt0,
                                                             const float* p1, uint32_t n1, void* w1, int dt1, int dh) {
  const bool second = blockIdx.y != 0;
  const float* p = second ? p1 : p0;
  const uint32_t n = second ? n1 : n0;
  void* w = second ? w1 : w0;
  const int dt = second ? dt1 : dt0;
  if (w == nullptr) return;
  __shared__ float red[16][17];
  const int cl = threadIdx.x & 15, rl = threadIdx.x >> 4, c = blockIdx.x * 16 + cl;
  float s = 0.f;
  if (c < dh)
    for (uint32_t i = rl; i < n; i += 16) s += p[(int64_t)i * dh + c];
  red[rl][cl] = s;
  __syncthreads();
  if (rl == 0 && c < dh) {
    s = 0.f;
    for (int i = 0; i < 16; ++i) s += red[i][cl];
    if (dt == HCLSM_F32) reinterpret_cast<float*>(w)[c] = s;
    else if (dt == HCLSM_BF16) reinterpret_cast<uint16_t*>(w)[c] = f32_to_bf16_bits(s);
    else reinterpret_cast<_Float16*>(w)[c] = (_Float16)s;
  }
}

namespace {

bool nr_aligned(const void* p, int64_t s0, int64_t s1, int64_t s2, int v, int esz) {
  return (uintptr_t)p % (uintptr_t)(v * esz) == 0 && s0 % v == 0 && s1 % v == 0 && s2 % v == 0;
}

int nr_check(const HclsmHeads* t, int bwd) {
  if (t->B < 0 || t->L < 0 || t->H < 0) return HCLSM_ERR_SHAPE;
  if (t->pos && t->pos_dtype != HCLSM_POS_I32 && t->pos_dtype != HCLSM_POS_I64) return HCLSM_ERR_DTYPE;
  if ((t->w || t->gw) && (t->w_dtype < HCLSM_F32 || t->w_dtype > HCLSM_F16)) return HCLSM_ERR_DTYPE;
  if (t->B > 0x7fffffff || t->L > 0x7fffffff || t->H > 0x7fffffff) return HCLSM_ERR_SHAPE;
  const int64_t chunks = (t->H + NR_HPL - 1) / NR_HPL;
  if (t->B && t->L && chunks && (t->B * t->L > 0x7fffffff / chunks)) return HCLSM_ERR_UNSUPPORTED;
  if (t->B && t->L && t->H && (t->x == nullptr || t->y == nullptr || (bwd && t->g == nullptr))) return HCLSM_ERR_NULL;
  return 0;
}

uint32_t nr_items(const HclsmHeads* t) { return (uint32_t)(t->B * t->L * ((t->H + NR_HPL - 1) / NR_HPL)); }

// Vector width: the widest of 16, 8, 4 (and 2) bytes at which every vector of a row starts on a boundary.
int nr_vec(const HclsmHeads* t, int n, int64_t dh, int64_t rot, int esz, int bwd) {
  for (int v = 16 / esz; v > 1; v >>= 1) {
    bool ok = rot % (2 * v) == 0 && dh % v == 0;
    for (int i = 0; i < n && ok; ++i) {
      if (nr_items(&t[i]) == 0) continue;
      ok = nr_aligned(t[i].x, t[i].x_sb, t[i].x_sl, t[i].x_sh, v, esz) && nr_aligned(t[i].y, 0, 0, 0, v, esz) &&
           (!bwd || nr_aligned(t[i].g, t[i].g_sb, t[i].g_sl, t[i].g_sh, v, esz));
    }
    if (ok) return v;
  }
  return 1;
}

template <int DT, int V, bool INTER>
void nr_launch(const NrArgs& a, int G, unsigned grid, int norm, int bwd, hipStream_t st) {
  constexpr int NU = V == 1 ? 2 : 1;   // 128 units of one pair at dh 256, at most 64 from V = 2 on
  if (bwd) hipLaunchKernelGGL((norm_rotary_kernel<DT, V, NU, INTER, true, true>), dim3(grid), dim3(NR_THREADS), 0, st, a, G);
  else if (norm) hipLaunchKernelGGL((norm_rotary_kernel<DT, V, NU, INTER, true, false>), dim3(grid), dim3(NR_THREADS), 0, st, a, G);
  else hipLaunchKernelGGL((norm_rotary_kernel<DT, V, NU, INTER, false, false>), dim3(grid), dim3(NR_THREADS), 0, st, a, G);
}

template <int DT, bool INTER>
void nr_launch_v(int v, const NrArgs& a, int G, unsigned grid, int norm, int bwd, hipStream_t st) {
  if constexpr (DT != HCLSM_F32) {
    if (v == 8) return nr_launch<DT, 8, INTER>(a, G, grid, norm, bwd, st);
  }
  if (v == 4) return nr_launch<DT, 4, INTER>(a, G, grid, norm, bwd, st);
  if (v == 2) return nr_launch<DT, 2, INTER>(a, G, grid, norm, bwd, st);
  return nr_launch<DT, 1, INTER>(a, G, grid, norm, bwd, st);
}

uint32_t nr_blocks(uint32_t items, int G, int bwd) {
  const uint32_t groups = NR_THREADS / G;
  const uint32_t n = items / groups + (items % groups != 0);
  const uint32_t most = bwd ? NR_BWD_BLOCKS : NR_FWD_BLOCKS;
  return n > most ? most : n;
}

int nr_run(const HclsmHeads* q, const HclsmHeads* k, int64_t dh, int64_t rot, int layout, const double* turns,
           float amp, float eps, int norm, int bwd, int dtype, float* ws, int64_t ws_bytes, hipStream_t st) {
  if (q == nullptr) return HCLSM_ERR_NULL;
  if (dtype < HCLSM_F32 || dtype > HCLSM_F16) return HCLSM_ERR_DTYPE;
  if (layout != HCLSM_ROTARY_HALF && layout != HCLSM_ROTARY_INTERLEAVED) return HCLSM_ERR_MODE;
  if (dh < 1 || rot < 0 || rot > dh || (rot & 1)) return HCLSM_ERR_SHAPE;
  if (dh > NR_MAX_DH) return HCLSM_ERR_UNSUPPORTED;
  if (rot > 0 && turns == nullptr) return HCLSM_ERR_NULL;
  HclsmHeads t[2] = {*q, k ? *k : HclsmHeads{}};
  const int n = k ? 2 : 1;
  for (int i = 0; i < n; ++i)
    if (int rc = nr_check(&t[i], bwd)) return rc;
  const int esz = dtype == HCLSM_F32 ? 4 : 2;
  const int v = nr_vec(t, n, dh, rot, esz, bwd);
  const int units = (int)((rot / 2) / v + (dh - rot + 2 * v - 1) / (2 * v));
  int G = 1;
  while (G < units && G < 64) G <<= 1;
  NrArgs a{};
  a.turns = turns;
  a.dh = (int)dh;
  a.rot = (int)rot;
  a.amp = amp;
  a.eps = eps;
  float* part = ws;
  for (int i = 0; i < n; ++i) {
    NrTensor& d = a.t[i];
    d.x = (const char*)t[i].x;
    d.g = (const char*)t[i].g;
    d.y = (char*)t[i].y;
    d.w = t[i].w;
    d.w_dtype = t[i].w_dtype;
    d.pos = t[i].pos;
    d.pos_dtype = t[i].pos_dtype;
    d.xsb = t[i].x_sb; d.xsl = t[i].x_sl; d.xsh = t[i].x_sh;
    d.gsb = t[i].g_sb; d.gsl = t[i].g_sl; d.gsh = t[i].g_sh;
    d.psb = t[i].pos_sb; d.psl = t[i].pos_sl;
    d.L = (uint32_t)t[i].L;
    d.H = (uint32_t)t[i].H;
    d.chunks = (uint32_t)((t[i].H + NR_HPL - 1) / NR_HPL);
    d.items = nr_items(&t[i]);
    d.blocks = nr_blocks(d.items, G, bwd);
    if (bwd && t[i].gw) {
      d.part = part;
      part += (int64_t)d.blocks * dh;
    }
  }
  if (bwd && (part - ws) * (int64_t)sizeof(float) > ws_bytes) return HCLSM_ERR_SHAPE;
  if (bwd && part != ws && ws == nullptr) return HCLSM_ERR_NULL;
  const unsigned grid = a.t[0].blocks + a.t[1].blocks;
  if (grid > 0) {
    const bool inter = layout == HCLSM_ROTARY_INTERLEAVED;
    if (dtype == HCLSM_F32) {
      if (inter) nr_launch_v<HCLSM_F32, true>(v, a, G, grid, norm, bwd, st);
      else nr_launch_v<HCLSM_F32, false>(v, a, G, grid, norm, bwd, st);
    } else if (dtype == HCLSM_BF16) {
      if (inter) nr_launch_v<HCLSM_BF16, true>(v, a, G, grid, norm, bwd, st);
      else nr_launch_v<HCLSM_BF16, false>(v, a, G, grid, norm, bwd, st);
    } else {
      if (inter) nr_launch_v<HCLSM_F16, true>(v, a, G, grid, norm, bwd, st);
      else nr_launch_v<HCLSM_F16, false>(v, a, G, grid, norm, bwd, st);
    }
    HCLSM_LAUNCH_CHECK();
  }
  if (bwd && (t[0].gw || t[1].gw)) {   // also for tensors without rows: their weights' gradient is zero
    hipLaunchKernelGGL(norm_rotary_dw_kernel, dim3((unsigned)((dh + 15) / 16), (unsigned)n), dim3(256), 0, st,
                       a.t[0].part, a.t[0].blocks, t[0].gw, t[0].w_dtype, a.t[1].part, a.t[1].blocks, t[1].gw,
                       t[1].w_dtype, (int)dh);
    HCLSM_LAUNCH_CHECK();
  }
  return 0;
}

}  // namespace
}  // namespace hclsm

extern "C" int hclsm_norm_rotary_forward(const HclsmHeads* q, const HclsmHeads* k, int64_t dh, int64_t rot, int layout,
                                         const double* turns, float amplitude, float eps, int norm, int dtype,
                                         void* stream) {
  return hclsm::nr_run(q, k, dh, rot, layout, turns, amplitude, eps, norm != 0, 0, dtype, nullptr, 0,
                       (hipStream_t)stream);
}

extern "C" int64_t hclsm_norm_rotary_backward_workspace(int64_t dh, int n_tensors) {
  if (dh < 1 || dh > hclsm::NR_MAX_DH || n_tensors < 1 || n_tensors > 2) return HCLSM_ERR_SHAPE;
  return (int64_t)n_tensors * hclsm::NR_BWD_BLOCKS * dh * (int64_t)sizeof(float);
}

extern "C" int hclsm_norm_rotary_backward(const HclsmHeads* q, const HclsmHeads* k, int64_t dh, int64_t rot, int layout,
                                          const double* turns, float amplitude, float eps, int dtype, void* workspace,
                                          int64_t workspace_bytes, void* stream) {
  return hclsm::nr_run(q, k, dh, rot, layout, turns, amplitude, eps, 1, 1, dtype, (float*)workspace, workspace_bytes,
                       (hipStream_t)stream);
}
