// Root-mean-square norm with the residual's addition, forward (in the input's type or in 8 bits) and backward (gfx950).
//
//     h = x + r (the stream, rounded to its type),  i = rsqrt(mean(h^2) + eps),  n = h i,  y = n w
//     dh = gh + i (gy w - n mean(gy w n)),  dx = dr = dh,  dw = sum over rows of gy n
//     8 bits: scale = max(max |y|, 2^-100) / 448 of a row or of each group of columns, y8 = y / scale rounded to e4m3
// The norm is that of the stream as it is written, as a program that adds and then normalises has it; the backward reads it
// back and needs no other of the forward's values.  Everything between a load and the one rounding at the store is float32.
//
// What bounds it: HBM.  A row is held in registers by TPR threads, U vectors of V elements each (16 bytes of x; single
// elements where the columns or the alignment do not allow it), so that it is read once; the weight stays in registers while a
// workgroup goes from row to row, the next row's loads in flight.  The backward's two sums travel together.
// Measured, bf16: 50176 x 384 forward 29 us, backward 28 and dw's sums 4 (5.0 TB/s together); 32768 x 4096 to 8 bits 185 us,
// 5.1 TB/s; 64 x 768 3.5 us (latency).  8027 x 1001 in single elements, float16 with a float32 stream: forward 21 us, backward 26,
// 4.4 TB/s.  A copy of 1 GiB reaches 5.04.
#include "internal.h"

namespace hclsm {

constexpr int RN_MAX_D = 16384;
constexpr int RN_BWD_BLOCKS = 1024;   // most workgroups (= partial sums of dw) of the backward
constexpr int RN_FWD_WAVES = 256 * 32;   // waves of a forward launch: the chip's places, the rows looped over
constexpr float RN_E4M3_MAX = 448.f;
constexpr float RN_LEAST = 0x1p-100f;    // smallest maximum that a scale is made for
enum { RN_FWD, RN_FP8, RN_BWD };

struct RnArgs {
  const char *x, *r, *h, *gy, *gh;    // r, gh nullable; h: the stream (backward)
  int64_t xs, rs, hs, gys, ghs;       // element strides of rows
  const void* w;                      // [D] or null (ones)
  char *y, *ho;                       // contiguous [rows, D]; ho null: not written
  char *dx, *dr;                      // contiguous; dr null: not written (the same as dx, or not wanted)
  float* scale;                       // [rows, D / group]
  float* part;                        // [blocks][D] partial sums of dw, null when not wanted
  int64_t rows;
  int D, group, w_dtype;              // group 0: a scale for the whole row
  float eps, inv_d;
};

__device__ __forceinline__ float rn_weight(const void* w, int dt, int i) {
  if (w == nullptr) return 1.f;
  if (dt == HCLSM_F32) return reinterpret_cast<const float*>(w)[i];
  if (dt == HCLSM_BF16) return bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(w)[i]);
  return (float)reinterpret_cast<const _Float16*>(w)[i];
}

// V consecutive elements as whole vectors of up to 16 bytes.
template <int DT, int V> struct RnVec {
  using E = typename Elem<DT>::T;
  static constexpr int BYTES = V * (int)sizeof(E), N = BYTES >= 16 ? BYTES / 16 : 1;
  uint4 w[N];
  __device__ __forceinline__ void load(const char* base, int64_t i) {
    const E* p = reinterpret_cast<const E*>(base) + i;
    if constexpr (BYTES >= 16) {
#pragma unroll
      for (int k = 0; k < N; ++k) w[k] = reinterpret_cast<const uint4*>(p)[k];
    } else {
      static_assert(V == 1, "16 bytes or one element");
      if constexpr (sizeof(E) == 4) w[0].x = __float_as_uint(*reinterpret_cast<const float*>(p));
      else w[0].x = *reinterpret_cast<const uint16_t*>(p);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int k = 0; k < N; ++k) w[k] = uint4{0, 0, 0, 0};
  }
  __device__ __forceinline__ void unpack(float* f) const {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const uint32_t q[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
      constexpr int PER = sizeof(E) == 4 ? 4 : 8;
#pragma unroll
      for (int i = 0; i < (V < PER ? V : PER); ++i) {
        if constexpr (DT == HCLSM_F32) f[k * PER + i] = __uint_as_float(q[i]);
        else if constexpr (DT == HCLSM_BF16) f[k * PER + i] = i & 1 ? __uint_as_float(q[i >> 1] & 0xffff0000u) : __uint_as_float(q[i >> 1] << 16);
        else f[k * PER + i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(q[i >> 1] >> (16 * (i & 1))));
      }
    }
  }
  __device__ __forceinline__ void pack(const float* f) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      uint32_t q[4] = {0, 0, 0, 0};
      constexpr int PER = sizeof(E) == 4 ? 4 : 8;
#pragma unroll
      for (int i = 0; i < (V < PER ? V : PER); ++i) {
        if constexpr (DT == HCLSM_F32) q[i] = __float_as_uint(f[k * PER + i]);
        else if constexpr (DT == HCLSM_BF16) {
          if (V == 1) q[0] = f32_to_bf16_bits(f[i]);
          else if (!(i & 1)) q[i >> 1] = pack_bf16x2(f[k * PER + i], f[k * PER + i + 1]);
        } else {
          q[i >> 1] |= (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[k * PER + i]) << (16 * (i & 1));
        }
      }
      w[k] = uint4{q[0], q[1], q[2], q[3]};
    }
  }
  __device__ __forceinline__ void store(char* base, int64_t i) const {
    E* p = reinterpret_cast<E*>(base) + i;
    if constexpr (BYTES >= 16) {
#pragma unroll
      for (int k = 0; k < N; ++k) reinterpret_cast<uint4*>(p)[k] = w[k];
    } else if constexpr (sizeof(E) == 4) {
      *reinterpret_cast<uint32_t*>(p) = w[0].x;
    } else {
      *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0].x;
    }
  }
};

template <int CTRL> __device__ __forceinline__ float rn_dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}

// Sum over a wave, the same bits in every lane: within quads, halves and rows of 16 lanes, then rows.
__device__ __forceinline__ float rn_wave_sum(float v) {
  v += rn_dpp<0xb1>(v);       // quad_perm [1, 0, 3, 2]
  v += rn_dpp<0x4e>(v);       // quad_perm [2, 3, 0, 1]
  v += rn_dpp<0x141>(v);      // row_half_mirror
  v += rn_dpp<0x140>(v);      // row_mirror
  return rows4_sum(v);
}
// Maximum over the aligned groups of G lanes (a power of two); passes NaN on.
__device__ __forceinline__ float rn_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float rn_lane_max(float v, int G) {
  if (G > 1) v = rn_max(v, rn_dpp<0xb1>(v));
  if (G > 2) v = rn_max(v, rn_dpp<0x4e>(v));
  if (G > 4) v = rn_max(v, rn_dpp<0x141>(v));
  if (G > 8) v = rn_max(v, rn_dpp<0x140>(v));
  if (G > 16) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = rn_max(__uint_as_float(a[0]), __uint_as_float(a[1]));
  }
  if (G > 32) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = rn_max(__uint_as_float(a[0]), __uint_as_float(a[1]));
  }
  return v;
}

// DX: type of x, y and gy; DS: type of the stream.  A workgroup of NT threads holds NT / TPR rows at once.
template <int DX, int DS, int V, int U, int TPR, int MODE>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) rn_kernel(const RnArgs a) {
  constexpr int NT = TPR > 256 ? TPR : 256, RPB = NT / TPR, WPR = TPR / 64;
  using VX = RnVec<DX, V>;
  using VS = RnVec<DS, V>;
  __shared__ float red[2][RPB][WPR][2];
  __shared__ float top[2][RPB][WPR];
  const int tid = threadIdx.x % TPR, rg = threadIdx.x / TPR, wave = tid >> 6;
  int parity = 0;
  // both sums over a row's threads
  auto sums = [&](float& p, float& q) __attribute__((always_inline)) {
    p = rn_wave_sum(p);
    if (MODE == RN_BWD) q = rn_wave_sum(q);
    if constexpr (WPR > 1) {      // two sets in turn: a set is written again only behind the next barrier
      if ((tid & 63) == 0) {
        red[parity][rg][wave][0] = p;
        if (MODE == RN_BWD) red[parity][rg][wave][1] = q;
      }
      __syncthreads();
      p = q = 0.f;
#pragma unroll
      for (int i = 0; i < WPR; ++i) {
        p += red[parity][rg][i][0];
        if (MODE == RN_BWD) q += red[parity][rg][i][1];
      }
    }
  };

  int col[U];
  float w[U][V];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    col[k] = (tid + k * TPR) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) w[k][e] = col[k] < a.D ? rn_weight(a.w, a.w_dtype, col[k] + e) : 0.f;
  }
  float gw[MODE == RN_BWD ? U : 1][V];
  if constexpr (MODE == RN_BWD) {
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) gw[k][e] = 0.f;
  }

  VX vx[U];      // x, or gy
  VS vs[U];      // r, or the stream
  VS vg[MODE == RN_BWD ? U : 1];      // gh
  auto load = [&](int64_t row) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < U; ++k) {
      vx[k].zero();
      vs[k].zero();
      if constexpr (MODE == RN_BWD) vg[k].zero();
      if (row < a.rows && col[k] < a.D) {
        if constexpr (MODE == RN_BWD) {
          if (a.gy) vx[k].load(a.gy, row * a.gys + col[k]);
          vs[k].load(a.h, row * a.hs + col[k]);
          if (a.gh) vg[k].load(a.gh, row * a.ghs + col[k]);
        } else {
          vx[k].load(a.x, row * a.xs + col[k]);
          if (a.r) vs[k].load(a.r, row * a.rs + col[k]);
        }
      }
    }
  };
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t row = (int64_t)blockIdx.x * RPB + rg;
  load(row);
  for (int64_t first = (int64_t)blockIdx.x * RPB; first < a.rows; first += step, row += step) {
    const bool in = row < a.rows;
    float f[U][V], s[U][V], gh[MODE == RN_BWD ? U : 1][V];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      vx[k].unpack(f[k]);
      vs[k].unpack(s[k]);
      if constexpr (MODE == RN_BWD) vg[k].unpack(gh[k]);
    }
    if (first + step < a.rows) load(row + step);
    float p = 0.f, q = 0.f;
    if constexpr (MODE == RN_BWD) {
#pragma unroll
      for (int k = 0; k < U; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          p += s[k][e] * s[k][e];
          q += f[k][e] * w[k][e] * s[k][e];
        }
      sums(p, q);
      const float inv = rsqrtf(p * a.inv_d + a.eps), dot = q * inv * a.inv_d;
#pragma unroll
      for (int k = 0; k < U; ++k) {
        float d[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float n = s[k][e] * inv;
          gw[k][e] += in ? f[k][e] * n : 0.f;      // (a row that is not there has n = 0, but an infinite inv without eps)
          d[e] = gh[k][e] + inv * (f[k][e] * w[k][e] - n * dot);
        }
        if (in && col[k] < a.D) {
          VX o;
          o.pack(d);
          if (a.dx) o.store(a.dx, row * a.D + col[k]);
          if (a.dr) {
            VS t;
            t.pack(d);
            t.store(a.dr, row * a.D + col[k]);
          }
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (a.r) {
          VS t;
#pragma unroll
          for (int e = 0; e < V; ++e) f[k][e] += s[k][e];
          t.pack(f[k]);
          t.unpack(f[k]);
          if (a.ho && in && col[k] < a.D) t.store(a.ho, row * a.D + col[k]);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) p += f[k][e] * f[k][e];
      }
      sums(p, q);
      const float inv = rsqrtf(p * a.inv_d + a.eps);
#pragma unroll
      for (int k = 0; k < U; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) f[k][e] = f[k][e] * inv * w[k][e];
      if constexpr (MODE == RN_FWD) {
#pragma unroll
        for (int k = 0; k < U; ++k)
          if (in && col[k] < a.D) {
            VX o;
            o.pack(f[k]);
            o.store(a.y, row * a.D + col[k]);
          }
      } else {
        float m[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
          m[k] = 0.f;
          if (col[k] < a.D) {
#pragma unroll
            for (int e = 0; e < V; ++e) m[k] = rn_max(m[k], fabsf(f[k][e]));
          }
        }
        if (a.group) {
#pragma unroll
          for (int k = 0; k < U; ++k) m[k] = rn_lane_max(m[k], a.group / V);
        } else {
          float all = m[0];
#pragma unroll
          for (int k = 1; k < U; ++k) all = rn_max(all, m[k]);
          all = rn_lane_max(all, 64);
          if constexpr (WPR > 1) {
            if ((tid & 63) == 0) top[parity][rg][wave] = all;
            __syncthreads();
            all = top[parity][rg][0];
#pragma unroll
            for (int i = 1; i < WPR; ++i) all = rn_max(all, top[parity][rg][i]);
          }
#pragma unroll
          for (int k = 0; k < U; ++k) m[k] = all;
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
          const float scale = rn_max(m[k], RN_LEAST) / RN_E4M3_MAX, up = 1.f / scale;
          if (in && col[k] < a.D) {
            if constexpr (V == 1) {
              a.y[row * a.D + col[k]] = (char)__builtin_amdgcn_cvt_pk_fp8_f32(f[k][0] * up, 0.f, 0, false);
            } else {
              uint32_t o[V / 4];
#pragma unroll
              for (int e = 0; e < V / 4; ++e) {
                int t = __builtin_amdgcn_cvt_pk_fp8_f32(f[k][4 * e] * up, f[k][4 * e + 1] * up, 0, false);
                o[e] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[k][4 * e + 2] * up, f[k][4 * e + 3] * up, t, true);
              }
              if constexpr (V == 8) *reinterpret_cast<uint2*>(a.y + row * a.D + col[k]) = uint2{o[0], o[1]};
              else *reinterpret_cast<uint32_t*>(a.y + row * a.D + col[k]) = o[0];
            }
            if (a.group ? col[k] % a.group == 0 : col[k] == 0)
              a.scale[a.group ? row * (a.D / a.group) + col[k] / a.group : row] = scale;
          }
        }
      }
    }
    parity ^= 1;
  }

  if constexpr (MODE == RN_BWD) {
    // dw of this workgroup: its rows' sums added in order
    if (a.part == nullptr) return;
    if constexpr (RPB > 1) {
      __shared__ float acc[RPB - 1][TPR * U * V];
      if (rg > 0) {
#pragma unroll
        for (int k = 0; k < U; ++k)
#pragma unroll
          for (int e = 0; e < V; ++e) acc[rg - 1][(k * V + e) * TPR + tid] = gw[k][e];
      }
      __syncthreads();
      if (rg == 0) {
        for (int i = 0; i < RPB - 1; ++i)
#pragma unroll
          for (int k = 0; k < U; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) gw[k][e] += acc[i][(k * V + e) * TPR + tid];
      }
    }
    if (rg == 0) {
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (col[k] < a.D)
#pragma unroll
          for (int e = 0; e < V; ++e) a.part[(int64_t)blockIdx.x * a.D + col[k] + e] = gw[k][e];
    }
  }
}

// dw[c] = sum over the workgroups of part[.][c], in a fixed order: 16 columns x 64 row lanes per workgroup.
__global__ void __launch_bounds__(1024) rn_dw_kernel(const float* part, int n, void* w, int dt, int D) {
  __shared__ float red[64][17];
  const int cl = threadIdx.x & 15, rl = threadIdx.x >> 4, c = blockIdx.x * 16 + cl;
  float s = 0.f;
  if (c < D) {
    for (int i = rl; i < n; i += 64 * 8) {       // the loads of eight rows in flight
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = i + 64 * j < n ? part[(int64_t)(i + 64 * j) * D + c] : 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[j];
    }
  }
  red[rl][cl] = s;
  __syncthreads();
  if (rl == 0 && c < D) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 64; ++i) s += red[i][cl];
    if (dt == HCLSM_F32) reinterpret_cast<float*>(w)[c] = s;
    else if (dt == HCLSM_BF16) reinterpret_cast<uint16_t*>(w)[c] = f32_to_bf16_bits(s);
    else reinterpret_cast<_Float16*>(w)[c] = (_Float16)s;
  }
}

namespace {

// Threads of a row and vectors of a thread: one vector each, the fewest threads of 64, 128, 256, 512 and 1024.  More vectors to fewer
// threads, bf16: 64 x 768 4.1 us by two to 64 threads, 3.5 by one to 128; 8192 x 4096 58.2 by two to 256, 54.5 by one to 512;
// 8192 x 8192 106.5 by four to 256, 101 by one to 1024, backward 132 and 121, 8 bits 101 and 92.  More threads than it takes: 50176 x
// 384 30.5 by one to 64, 37.7 to 256; 32768 x 768 backward 37 by one to 128, 45 to 256 (42 by two to 64).
// Longer rows do not fit the 128 registers of 1024 threads in the backward, and the compiler spills (bytes a lane): two vectors 48 (bf16), 36
// (float16), 168 (float32 stream), four of float32 204, 16 single elements 228 to 240, and 36 to 44 in their 8-bit form.  67 million elements,
// backward by rows of 8192 and 16384: bf16 124 and 180 us, float32 stream 225 and 444, float32 225 and 427; by rows of 5001, backward 770 to
// 1040, 8 bits 290 to 360, forward (without spills) 157 to 214.  Forward and 8 bits of 16384 run as shorter rows do, 4.8 to 5.2 TB/s.
struct RnShape {
  int tpr, u;
};
RnShape rn_shape(int64_t D, int v) {
  if (v == 1) return D <= 256 ? RnShape{64, 4} : D <= 1024 ? RnShape{256, 4} : D <= 4096 ? RnShape{1024, 4} : RnShape{1024, 16};
  const int64_t n = (D + v - 1) / v;
  return n <= 64 ? RnShape{64, 1} : n <= 128 ? RnShape{128, 1} : n <= 256 ? RnShape{256, 1} : n <= 512 ? RnShape{512, 1} : n <= 1024 ? RnShape{1024, 1}
         : n <= 2048 ? RnShape{1024, 2} : RnShape{1024, 4};
}
int64_t rn_blocks(int64_t rows, int tpr, int mode) {
  const int64_t rpb = tpr < 256 ? 256 / tpr : 1, n = (rows + rpb - 1) / rpb;
  const int64_t most = mode == RN_BWD ? RN_BWD_BLOCKS : RN_FWD_WAVES / (tpr > 256 ? tpr / 64 : 4);
  return n > most ? most : n;
}

template <int DX, int DS, int V, int U, int TPR> void rn_launch_m(const RnArgs& a, int mode, unsigned grid, hipStream_t st) {
  const dim3 gr(grid), bl(TPR > 256 ? TPR : 256);
  if (mode == RN_FWD) hipLaunchKernelGGL((rn_kernel<DX, DS, V, U, TPR, RN_FWD>), gr, bl, 0, st, a);
  else if (mode == RN_FP8) hipLaunchKernelGGL((rn_kernel<DX, DS, V, U, TPR, RN_FP8>), gr, bl, 0, st, a);
  else hipLaunchKernelGGL((rn_kernel<DX, DS, V, U, TPR, RN_BWD>), gr, bl, 0, st, a);
}

template <int DX, int DS> void rn_launch(const RnArgs& a, int v, RnShape s, int mode, unsigned grid, hipStream_t st) {
  constexpr int V = DX == HCLSM_F32 ? 4 : 8;
  if (v == 1) {
    if (s.tpr == 64) rn_launch_m<DX, DS, 1, 4, 64>(a, mode, grid, st);
    else if (s.tpr == 256) rn_launch_m<DX, DS, 1, 4, 256>(a, mode, grid, st);
    else if (s.u == 4) rn_launch_m<DX, DS, 1, 4, 1024>(a, mode, grid, st);
    else rn_launch_m<DX, DS, 1, 16, 1024>(a, mode, grid, st);
  } else if (s.tpr == 64) {
    rn_launch_m<DX, DS, V, 1, 64>(a, mode, grid, st);
  } else if (s.tpr == 128) {
    rn_launch_m<DX, DS, V, 1, 128>(a, mode, grid, st);
  } else if (s.tpr == 256) {
    rn_launch_m<DX, DS, V, 1, 256>(a, mode, grid, st);
  } else if (s.tpr == 512) {
    rn_launch_m<DX, DS, V, 1, 512>(a, mode, grid, st);
  } else if (s.u == 1) {
    rn_launch_m<DX, DS, V, 1, 1024>(a, mode, grid, st);
  } else if (s.u == 2) {
    rn_launch_m<DX, DS, V, 2, 1024>(a, mode, grid, st);
  } else if constexpr (V == 4) {
    rn_launch_m<DX, DS, V, 4, 1024>(a, mode, grid, st);
  }
}

bool rn_aligned(const void* p, int64_t stride, int dtype) {
  return (uintptr_t)p % 16 == 0 && stride % (dtype == HCLSM_F32 ? 4 : 8) == 0;
}

int rn_sizes(int64_t rows, int64_t D, int dtype, int stream_dtype) {
  if (rows < 0 || D < 1) return HCLSM_ERR_SHAPE;
  if (dtype < HCLSM_F32 || dtype > HCLSM_F16 || (stream_dtype != dtype && stream_dtype != HCLSM_F32)) return HCLSM_ERR_DTYPE;
  if (D > RN_MAX_D || rows > ((int64_t)1 << 40)) return HCLSM_ERR_UNSUPPORTED;
  return 0;
}

int rn_run(const HclsmResidualNorm* x, int mode, void* ws, int64_t ws_bytes, hipStream_t st) {
  if (x == nullptr) return HCLSM_ERR_NULL;
  if (int rc = rn_sizes(x->rows, x->D, x->dtype, x->stream_dtype)) return rc;
  if ((x->w || x->dw) && (x->w_dtype < HCLSM_F32 || x->w_dtype > HCLSM_F16)) return HCLSM_ERR_DTYPE;
  if (!(x->eps >= 0.f)) return HCLSM_ERR_SHAPE;
  if (mode == RN_FP8 && x->group != 0 && x->group != 32 && x->group != 64 && x->group != 128) return HCLSM_ERR_UNSUPPORTED;
  if (mode == RN_FP8 && x->group != 0 && x->D % x->group) return HCLSM_ERR_SHAPE;
  const bool bwd = mode == RN_BWD;
  const int esz = x->dtype == HCLSM_F32 ? 4 : 2, v0 = 16 / esz;
  RnArgs a{};
  a.x = (const char*)x->x; a.r = (const char*)x->r; a.h = (const char*)x->h; a.gy = (const char*)x->gy; a.gh = (const char*)x->gh;
  a.xs = x->x_sr; a.rs = x->r_sr; a.hs = x->h_sr; a.gys = x->gy_sr; a.ghs = x->gh_sr;
  a.w = x->w; a.w_dtype = x->w_dtype;
  a.y = (char*)x->y; a.ho = (char*)x->h_out;
  a.dx = (char*)x->dx; a.dr = (char*)x->dr;
  a.scale = x->scale;
  a.rows = x->rows; a.D = (int)x->D; a.group = (int)x->group;
  a.eps = x->eps; a.inv_d = 1.f / (float)x->D;
  if (x->rows > 0) {
    if (bwd ? !x->h : !x->x || !x->y || (mode == RN_FP8 && !x->scale)) return HCLSM_ERR_NULL;
  }
  const int sd = x->stream_dtype;
  bool wide = x->D % v0 == 0;
  for (const void* p : {x->x, x->r, x->h, x->gy, x->gh, (const void*)x->y, (const void*)x->h_out, (const void*)x->dx,
                        (const void*)x->dr}) wide = wide && (uintptr_t)p % 16 == 0;
  if (x->rows > 1) {
    wide = wide && (bwd ? (!x->gy || rn_aligned(x->gy, x->gy_sr, x->dtype)) && rn_aligned(x->h, x->h_sr, sd) &&
                              (!x->gh || rn_aligned(x->gh, x->gh_sr, sd))
                        : rn_aligned(x->x, x->x_sr, x->dtype) && (!x->r || rn_aligned(x->r, x->r_sr, sd)));
    // a float32 stream is read in twice as many vectors; its rows are on 16-byte boundaries where those of x are
  }
  const int v = wide ? v0 : 1;
  if (mode == RN_FP8 && x->group != 0 && v == 1) return HCLSM_ERR_UNSUPPORTED;
  const RnShape s = rn_shape(x->D, v);
  const int64_t blocks = rn_blocks(x->rows, s.tpr, mode);
  if (bwd && x->dw) {
    if (ws == nullptr) return HCLSM_ERR_NULL;
    if (ws_bytes < blocks * x->D * 4) return HCLSM_ERR_SHAPE;
    if ((uintptr_t)ws % 16) return HCLSM_ERR_UNSUPPORTED;
    a.part = (float*)ws;
  }
  if (blocks > 0) {
    const unsigned g = (unsigned)blocks;
    if (x->dtype == HCLSM_F32) rn_launch<HCLSM_F32, HCLSM_F32>(a, v, s, mode, g, st);
    else if (x->dtype == HCLSM_BF16 && sd == HCLSM_BF16) rn_launch<HCLSM_BF16, HCLSM_BF16>(a, v, s, mode, g, st);
    else if (x->dtype == HCLSM_BF16) rn_launch<HCLSM_BF16, HCLSM_F32>(a, v, s, mode, g, st);
    else if (sd == HCLSM_F16) rn_launch<HCLSM_F16, HCLSM_F16>(a, v, s, mode, g, st);
    else rn_launch<HCLSM_F16, HCLSM_F32>(a, v, s, mode, g, st);
    HCLSM_LAUNCH_CHECK();
  }
  if (bwd && x->dw) {      // also without rows: a gradient of zeros
    hipLaunchKernelGGL(rn_dw_kernel, dim3((unsigned)((x->D + 15) / 16)), dim3(1024), 0, st, a.part, (int)blocks, x->dw, x->w_dtype,
                       (int)x->D);
    HCLSM_LAUNCH_CHECK();
  }
  return 0;
}

}  // namespace
}  // namespace hclsm

extern "C" int hclsm_residual_norm_forward(const HclsmResidualNorm* x, void* stream) {
  return hclsm::rn_run(x, hclsm::RN_FWD, nullptr, 0, (hipStream_t)stream);
}

extern "C" int hclsm_residual_norm_fp8(const HclsmResidualNorm* x, void* stream) {
  return hclsm::rn_run(x, hclsm::RN_FP8, nullptr, 0, (hipStream_t)stream);
}

extern "C" int64_t hclsm_residual_norm_backward_workspace(int64_t rows, int64_t D) {
  using namespace hclsm;
  if (int rc = rn_sizes(rows, D, HCLSM_F32, HCLSM_F32)) return rc;
  // whatever the vectors' width
  return (rows < RN_BWD_BLOCKS ? rows : RN_BWD_BLOCKS) * D * 4;
}

extern "C" int hclsm_residual_norm_backward(const HclsmResidualNorm* x, void* workspace, int64_t workspace_bytes, void* stream) {
  return hclsm::rn_run(x, hclsm::RN_BWD, workspace, workspace_bytes, (hipStream_t)stream);
}
