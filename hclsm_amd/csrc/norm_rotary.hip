// Norms of queries and keys for each head and their position rotation, forward and backward (gfx950).
//
// One row is one head of one token: dh elements x.  With r = rsqrt(mean(x^2) + eps) (1 without the norm) and the
// weight w (1 without one),
//     n = x r,   y = R(n w),
// where R turns pair i (elements (i, i + rot/2) or (2i, 2i + 1) of the first rot) by position * frequency_i and
// scales it by an amplitude; elements from rot on pass through.  R^T, which turns back, gives the gradients:
//     d = R^T g,   dw = sum over rows of d n,   dx = r (d w - n mean(d w n)).
// Everything between the load and the one rounding at the store is float32, but for the angle: it is formed in turns,
// t = position * (frequency / 2 pi), in float64, and only what is left of t after its whole and quarter turns is rounded to
// float32, as an angle: a position of 2^31 still leaves 2^-22 turns.
//
// What bounds it: HBM.  A row is spread over G lanes that hold V pairs each: two vectors of V elements per lane and row,
// V = 4 where rot, dh, the strides and the addresses allow it (16 B loads of float32, 8 B of 16-bit elements), else 2 or 1.
// 16-byte loads of 16-bit elements would halve the lanes and double what each keeps (weights, their gradients, angles):
// 52 -> 73 us for the backward below, 36 -> 41 us for its forward.  A lane group takes a token's heads one after another,
// the next loads in flight, so that an angle (about 40 instructions, some in float64) serves all of them; where the tokens
// alone do not fill the chip, a token's heads are shared by several groups.
// Measured (bf16, 32 x 1568 tokens, 6 + 6 heads of 64): forward 35 us and backward 52 us, 4.4 TB/s of the bytes that have to
// move, against 5.1 TB/s of a 1 GiB copy; the sum of the weights' gradient 4 us; rotation of 12 heads of 32 x 1024 tokens
// 22 us, 4.5 TB/s.
#include "internal.h"

namespace hclsm {

constexpr int NR_THREADS = 256;
constexpr int NR_HPL = 2;             // heads of a token that a lane group works on at once (backward: one)
constexpr int NR_MAX_DH = 256;
constexpr int NR_BWD_BLOCKS = 1024;   // most workgroups (= partial sums of dw) per tensor of the backward
constexpr int NR_FILL_WAVES = 256 * 4 * 4;   // waves that keep every SIMD's loads in flight
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
  uint32_t L, H;
  uint32_t chunks, hpi;         // a token's heads are shared by `chunks` items of hpi heads each
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
  W w;
  __device__ __forceinline__ void load(const E* p) { w = *reinterpret_cast<const W*>(p); }
  __device__ __forceinline__ void store(E* p) const { *reinterpret_cast<W*>(p) = w; }
  __device__ __forceinline__ void unpack(float* f) const {
    if constexpr (DT == HCLSM_F32 || V == 1) {
      struct A { E e[V]; } a = __builtin_bit_cast(A, w);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = Elem<DT>::ld(&a.e[i]);
    } else {
      struct A { uint32_t u[V / 2]; } a = __builtin_bit_cast(A, w);
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        if constexpr (DT == HCLSM_BF16) {
          f[2 * i] = __uint_as_float(a.u[i] << 16);
          f[2 * i + 1] = __uint_as_float(a.u[i] & 0xffff0000u);
        } else {
          f[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)a.u[i]);
          f[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(a.u[i] >> 16));
        }
      }
    }
  }
  __device__ __forceinline__ void pack(const float* f) {
    if constexpr (DT == HCLSM_F32 || V == 1) {
      struct A { E e[V]; } a;
#pragma unroll
      for (int i = 0; i < V; ++i) Elem<DT>::st(&a.e[i], f[i]);
      w = __builtin_bit_cast(W, a);
    } else {
      struct A { uint32_t u[V / 2]; } a;
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        if constexpr (DT == HCLSM_BF16) {
          a.u[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
        } else {
          typedef _Float16 h2 __attribute__((ext_vector_type(2)));
          a.u[i] = __builtin_bit_cast(uint32_t, h2{(_Float16)f[2 * i], (_Float16)f[2 * i + 1]});
        }
      }
      w = __builtin_bit_cast(W, a);
    }
  }
};

__device__ __forceinline__ float nr_weight(const void* w, int dt, int i) {
  if (w == nullptr) return 1.f;
  if (dt == HCLSM_F32) return reinterpret_cast<const float*>(w)[i];
  if (dt == HCLSM_BF16) return bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(w)[i]);
  return (float)reinterpret_cast<const _Float16*>(w)[i];
}

template <int CTRL> __device__ __forceinline__ float nr_dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}

// Sum over the G lanes of a group (G a power of two, groups aligned), the same bits in every lane: neighbours by
// permutations inside a row of 16 lanes (within a quad, then of mirrored halves), then rows and halves of the wave.
__device__ __forceinline__ float nr_group_sum(float v, int G) {
  if (G > 1) v += nr_dpp<0xb1>(v);       // quad_perm [1, 0, 3, 2]
  if (G > 2) v += nr_dpp<0x4e>(v);       // quad_perm [2, 3, 0, 1]
  if (G > 4) v += nr_dpp<0x141>(v);      // row_half_mirror
  if (G > 8) v += nr_dpp<0x140>(v);      // row_mirror
  if (G > 16) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  }
  if (G > 32) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  }
  return v;
}

// sin and cos of t turns, |t| <= 1/2: the nearest quarter turn taken off in float64 and the rest made an angle there, then in
// float32 the Taylor polynomials of degree 9 and 10 on at most an eighth of a turn (remainders below 2^-28) and the quarter
// turns put back by exchange and sign.  Off by at most 1.4 times 2^-24 (rms 1.2 times that of rounding the values to float32).
// About 20 instructions besides the four in float64; the library's sincospif takes twice that.
__device__ __forceinline__ void nr_sincos(double t, float& s, float& c) {
  const double t4 = 4.0 * t, q = rint(t4);
  const float x = (float)((t4 - q) * 1.57079632679489662), z = x * x;
  const int n = (int)q;
  const float sp = x + x * z * (-1.f / 6 + z * (1.f / 120 + z * (-1.f / 5040 + z * (1.f / 362880))));
  const float cp = 1.f + z * (-0.5f + z * (1.f / 24 + z * (-1.f / 720 + z * (1.f / 40320 - z * (1.f / 3628800)))));
  const float a = n & 1 ? cp : sp, b = n & 1 ? sp : cp;
  s = __uint_as_float(__float_as_uint(a) ^ ((uint32_t)(n & 2) << 30));
  c = __uint_as_float(__float_as_uint(b) ^ ((uint32_t)((n + 1) & 2) << 30));
}

// V: pairs per lane and unit.  NU: units per lane.  A unit is two vectors of V elements: unit u < rot / 2V holds pairs
// uV .. uV + V - 1 (INTER: elements 2uV .. 2uV + 2V - 1, else uV .. and rot/2 + uV ..), later units hold
// the elements that pass through, 2V each, the last one possibly V.
// FULL: rot = dh, every unit holds pairs.  Elsewhere units that pass through are selected, not turned by a zero angle:
// an infinity or NaN among them would reach its neighbour.
template <int DT, int V, int NU, bool INTER, bool NORM, bool BWD, bool FULL>
__global__ void __launch_bounds__(NR_THREADS) norm_rotary_kernel(NrArgs a, int G) {
  using E = typename Elem<DT>::T;
  using Vec = NrVec<DT, V>;
  constexpr int HPL = BWD ? 1 : NR_HPL;
  const float inv_dh = 1.f / (float)a.dh;
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
    const uint32_t first = c * t.hpi;
    const uint32_t end = !live ? first : first + t.hpi < t.H ? first + t.hpi : t.H;

    Vec xn[HPL][NU][2], gn[BWD ? HPL : 1][NU][2];
    auto load = [&](uint32_t h0) __attribute__((always_inline)) {
      const int nh = h0 >= end ? 0 : (int)(end - h0 < HPL ? end - h0 : HPL);
      const E* xp = reinterpret_cast<const E*>(t.x) + b * t.xsb + l * t.xsl + h0 * t.xsh;
      const E* gp = BWD ? reinterpret_cast<const E*>(t.g) + b * t.gsb + l * t.gsl + h0 * t.gsh : nullptr;
#pragma unroll
      for (int h = 0; h < HPL; ++h)
#pragma unroll
        for (int k = 0; k < NU; ++k)
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            xn[h][k][s] = Vec{};
            if (BWD) gn[h][k][s] = Vec{};
            if (h < nh && col[k][s] >= 0) {
              xn[h][k][s].load(xp + h * t.xsh + col[k][s]);
              if (BWD) gn[h][k][s].load(gp + h * t.gsh + col[k][s]);
            }
          }
    };
    load(first);

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
          nr_sincos(tr, sn[k][j], cs[k][j]);
          sn[k][j] *= a.amp;
          cs[k][j] *= a.amp;
        }
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) { cs[k][j] = 1.f; sn[k][j] = 0.f; }
      }
    }

    // the whole group takes the same number of rounds (the sums need every lane)
    for (uint32_t h0 = first; h0 < first + t.hpi; h0 += HPL) {
      const int nh = h0 >= end ? 0 : (int)(end - h0 < HPL ? end - h0 : HPL);
      Vec x[HPL][NU][2], g[BWD ? HPL : 1][NU][2];
#pragma unroll
      for (int h = 0; h < HPL; ++h)
#pragma unroll
        for (int k = 0; k < NU; ++k)
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            x[h][k][s] = xn[h][k][s];
            if (BWD) g[h][k][s] = gn[h][k][s];
          }
      if (h0 + HPL < first + t.hpi) load(h0 + HPL);
      E* yp = reinterpret_cast<E*>(t.y) + ((int64_t)tok * t.H + h0) * a.dh;
#pragma unroll
      for (int h = 0; h < HPL; ++h) {
        if (NORM ? h0 + h >= first + t.hpi : h >= nh) continue;
        float xf[NU][2 * V], r = 1.f;
#pragma unroll
        for (int k = 0; k < NU; ++k) { x[h][k][0].unpack(xf[k]); x[h][k][1].unpack(xf[k] + V); }
        if (NORM) {
          float ss = 0.f;
#pragma unroll
          for (int k = 0; k < NU; ++k)
#pragma unroll
            for (int j = 0; j < 2 * V; ++j) ss += xf[k][j] * xf[k][j];
          r = rsqrtf(nr_group_sum(ss, G) * inv_dh + a.eps);
          r = h < nh ? r : 0.f;       // a head that is not there adds nothing to dw
        }
        float y[NU][2 * V];
        if (!BWD) {
#pragma unroll
          for (int k = 0; k < NU; ++k) {
            float e[2 * V];
#pragma unroll
            for (int j = 0; j < 2 * V; ++j) e[j] = NORM ? xf[k][j] * r * w[k][j] : xf[k][j];
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const int ia = INTER ? 2 * j : j, ib = INTER ? 2 * j + 1 : V + j;
              y[k][ia] = e[ia] * cs[k][j] - e[ib] * sn[k][j];
              y[k][ib] = e[ib] * cs[k][j] + e[ia] * sn[k][j];
              if (!FULL) {
                y[k][ia] = pair[k] ? y[k][ia] : e[ia];
                y[k][ib] = pair[k] ? y[k][ib] : e[ib];
              }
            }
          }
        } else {
          float gf[NU][2 * V], dot = 0.f;
#pragma unroll
          for (int k = 0; k < NU; ++k) {
            g[h][k][0].unpack(gf[k]);
            g[h][k][1].unpack(gf[k] + V);
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const int ia = INTER ? 2 * j : j, ib = INTER ? 2 * j + 1 : V + j;
              const float ga = gf[k][ia], gb = gf[k][ib];
              y[k][ia] = ga * cs[k][j] + gb * sn[k][j];
              y[k][ib] = gb * cs[k][j] - ga * sn[k][j];
              if (!FULL) {
                y[k][ia] = pair[k] ? y[k][ia] : ga;
                y[k][ib] = pair[k] ? y[k][ib] : gb;
              }
            }
#pragma unroll
            for (int j = 0; j < 2 * V; ++j) {
              xf[k][j] *= r;
              gw[k][j] += y[k][j] * xf[k][j];
              y[k][j] *= w[k][j];
              dot += y[k][j] * xf[k][j];
            }
          }
          dot = nr_group_sum(dot, G) * inv_dh;
#pragma unroll
          for (int k = 0; k < NU; ++k)
#pragma unroll
            for (int j = 0; j < 2 * V; ++j) y[k][j] = r * (y[k][j] - xf[k][j] * dot);
        }
        if (h < nh) {
#pragma unroll
          for (int k = 0; k < NU; ++k)
#pragma unroll
            for (int s = 0; s < 2; ++s)
              if (col[k][s] >= 0) {
                Vec o;
                o.pack(y[k] + s * V);
                o.store(yp + h * a.dh + col[k][s]);
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

// gw[c] = sum over blocks of part[block][c], in a fixed order: 16 columns x 64 row lanes per workgroup.
__global__ void __launch_bounds__(1024) norm_rotary_dw_kernel(const float* p0, uint32_t n0, void* w0, int dt0,
                                                              const float* p1, uint32_t n1, void* w1, int dt1, int dh) {
  const bool second = blockIdx.y != 0;
  const float* p = second ? p1 : p0;
  const uint32_t n = second ? n1 : n0;
  void* w = second ? w1 : w0;
  const int dt = second ? dt1 : dt0;
  if (w == nullptr) return;
  __shared__ float red[64][17];
  const int cl = threadIdx.x & 15, rl = threadIdx.x >> 4, c = blockIdx.x * 16 + cl;
  float s = 0.f;
  if (c < dh) {
    for (uint32_t i = rl; i < n; i += 64 * 8) {       // the loads of eight rows in flight
      float v[8];
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) v[j] = i + 64 * j < n ? p[(int64_t)(i + 64 * j) * dh + c] : 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[j];
    }
  }
  red[rl][cl] = s;
  __syncthreads();
  if (rl == 0 && c < dh) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 64; ++i) s += red[i][cl];
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
  const int64_t chunks = t->H;     // at most
  if (t->B && t->L && chunks && (t->B * t->L > 0x7fffffff / chunks)) return HCLSM_ERR_UNSUPPORTED;
  if (t->B && t->L && t->H && (t->x == nullptr || t->y == nullptr || (bwd && t->g == nullptr))) return HCLSM_ERR_NULL;
  return 0;
}

// Items of a token: one where the tokens alone fill the chip (an angle then serves all of a token's heads), otherwise
// up to one per `hpl` heads.
void nr_split(const HclsmHeads* t, int G, int hpl, uint32_t* chunks, uint32_t* hpi) {
  const int64_t tokens = t->B * t->L, most = (t->H + hpl - 1) / hpl;
  const int64_t fill = (int64_t)NR_FILL_WAVES * (64 / G);
  int64_t n = tokens > 0 ? (fill + tokens - 1) / tokens : 1;
  n = n > most ? most : n;
  n = n < 1 ? 1 : n;
  const int64_t per = (t->H + n - 1) / n;
  *hpi = (uint32_t)(per > 0 ? per : 1);
  *chunks = (uint32_t)((t->H + *hpi - 1) / *hpi);
}

// Vector width: the widest of 16, 8, 4 (and 2) bytes at which every vector of a row starts on a boundary.
int nr_vec(const HclsmHeads* t, int n, int64_t dh, int64_t rot, int esz, int bwd) {
  for (int v = 4; v > 1; v >>= 1) {
    bool ok = rot % (2 * v) == 0 && dh % v == 0;
    for (int i = 0; i < n && ok; ++i) {
      if (t[i].B * t[i].L * t[i].H == 0) continue;
      ok = nr_aligned(t[i].x, t[i].x_sb, t[i].x_sl, t[i].x_sh, v, esz) && nr_aligned(t[i].y, 0, 0, 0, v, esz) &&
           (!bwd || nr_aligned(t[i].g, t[i].g_sb, t[i].g_sl, t[i].g_sh, v, esz));
    }
    if (ok) return v;
  }
  return 1;
}

template <int DT, int V, bool INTER, bool FULL>
void nr_launch(const NrArgs& a, int G, unsigned grid, int norm, int bwd, hipStream_t st) {
  constexpr int NU = V == 1 ? 2 : 1;   // 128 units of one pair at dh 256, at most 64 from V = 2 on
  const dim3 gr(grid), bl(NR_THREADS);
  if (bwd) hipLaunchKernelGGL((norm_rotary_kernel<DT, V, NU, INTER, true, true, FULL>), gr, bl, 0, st, a, G);
  else if (norm) hipLaunchKernelGGL((norm_rotary_kernel<DT, V, NU, INTER, true, false, FULL>), gr, bl, 0, st, a, G);
  else hipLaunchKernelGGL((norm_rotary_kernel<DT, V, NU, INTER, false, false, FULL>), gr, bl, 0, st, a, G);
}

template <int DT, int V, bool INTER>
void nr_launch_f(const NrArgs& a, int G, unsigned grid, int norm, int bwd, hipStream_t st) {
  if (a.rot == a.dh) nr_launch<DT, V, INTER, true>(a, G, grid, norm, bwd, st);
  else nr_launch<DT, V, INTER, false>(a, G, grid, norm, bwd, st);
}

template <int DT, bool INTER>
void nr_launch_v(int v, const NrArgs& a, int G, unsigned grid, int norm, int bwd, hipStream_t st) {
  if (v == 4) return nr_launch_f<DT, 4, INTER>(a, G, grid, norm, bwd, st);
  if (v == 2) return nr_launch_f<DT, 2, INTER>(a, G, grid, norm, bwd, st);
  return nr_launch_f<DT, 1, INTER>(a, G, grid, norm, bwd, st);
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
    nr_split(&t[i], G, NR_HPL, &d.chunks, &d.hpi);
    d.items = (uint32_t)(t[i].B * t[i].L * d.chunks);
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
    hipLaunchKernelGGL(norm_rotary_dw_kernel, dim3((unsigned)((dh + 15) / 16), (unsigned)n), dim3(1024), 0, st,
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
