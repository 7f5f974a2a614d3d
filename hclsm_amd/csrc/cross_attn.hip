// Cross attention: argument checks and dispatch by element type.
#include "cross_attn.h"

namespace hclsm {

namespace {

// Workgroups that share a unit's n keys or rows: as many as fill `slots` workgroups, of `least` each or more.
int ca_split(int64_t workgroups, int64_t slots, int64_t n, int64_t least) {
  int64_t s = workgroups > 0 ? slots / workgroups : 1;
  s = s > n / least ? n / least : s;
  return (int)(s < 1 ? 1 : s > CA_MAX_SPLIT ? CA_MAX_SPLIT : s);
}

int64_t ca_row_bytes(int64_t dh, int dtype) { return ca_padded_dh(dh) * (dtype == HCLSM_F32 ? 4 : 2); }

}  // namespace

CaPlan ca_forward_plan(int64_t B, int64_t Lq, int64_t Lk, int64_t Hk, int64_t G, int64_t dh, int dtype) {
  const int64_t rows = Lq * G, units = B * Hk, bytes = ca_row_bytes(dh, dtype);
  CaPlan p{0, 1, 1};
  p.few = rows <= 16 && bytes <= CA_FEW1_BYTES ? 1 : rows <= 32 && bytes <= ca_few2_bytes(dtype) ? 2 : 0;
  const int64_t per = p.few ? 16 * p.few : ca_tile_rows(rows, bytes);
  // workgroups that are on the chip at once (registers: 4 to 1 a CU for few rows, 3 to 2 for many)
  const int64_t slots = p.few ? (bytes <= 64 ? 1024 : bytes <= 128 ? 768 : bytes <= 192 ? 512 : 256) : bytes <= 128 ? 768 : 512;
  p.nsplit = ca_split(units * ((rows + per - 1) / per), slots, Lk, p.few ? 256 : 128);
  return p;
}

CaPlan ca_backward_plan(int64_t B, int64_t Lq, int64_t Lk, int64_t Hk, int64_t G, int64_t dh, int dtype) {
  const int64_t rows = Lq * G, units = B * Hk, bytes = ca_row_bytes(dh, dtype);
  CaPlan p{0, 1, 1};
  if (rows <= 32 && bytes <= CA_FEW_BWD_BYTES) {
    p.few = 2;
    p.nsplit = ca_split(units, 512, Lk, 256);
    return p;
  }
  const int64_t slots = 512, pq = ca_tile_rows(rows, bytes), pk = ca_tile_rows(Lk, bytes);
  p.nsplit = ca_split(units * ((rows + pq - 1) / pq), slots, Lk, 128);
  p.nrows = ca_split(units * ((Lk + pk - 1) / pk), slots, rows, 128);
  return p;
}

int64_t ca_backward_bytes(const CaPlan& p, int64_t B, int64_t Lq, int64_t Lk, int64_t Hk, int64_t G, int64_t dh) {
  const int64_t units = B * Hk, rows = Lq * G;
  const int64_t dq = p.nsplit > 1 ? p.nsplit * units * rows * dh * 4 : 0;
  if (p.few) return dq;
  return (units * rows * 4 + 255) / 256 * 256 + dq + (p.nrows > 1 ? 2 * p.nrows * units * Lk * dh * 4 : 0);
}

// A row's partial results joined: weights exp2(lse_s - lse), one workgroup per row, TC lanes of four columns each and
// 256 / TC groups of lanes that take every so many of the splits; the groups add up in order.
template <int DT>
__global__ void __launch_bounds__(256) ca_join_kernel(const CaArgs a, int tc) {
  __shared__ float s_lse[CA_MAX_SPLIT];
  __shared__ caf4 s_acc[256];
  const int all = a.Lq * a.G;
  const int64_t stride = (int64_t)a.units * all;
  for (int64_t row = blockIdx.x; row < stride; row += gridDim.x) {
    if ((int)threadIdx.x < a.nsplit) s_lse[threadIdx.x] = a.part_lse[(int64_t)threadIdx.x * stride + row];
    __syncthreads();
    float top = -INFINITY, sum = 0.f;
    for (int s = 0; s < a.nsplit; ++s) top = fmaxf(top, s_lse[s]);
    const float base = top == -INFINITY ? 0.f : top;
    for (int s = 0; s < a.nsplit; ++s) sum += fast_exp2(s_lse[s] - base);
    const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    const int c = threadIdx.x & (tc - 1), sl = threadIdx.x / tc, n = 256 / tc;
    caf4 acc = {0.f, 0.f, 0.f, 0.f};
    if (4 * c < a.dh) {
#pragma unroll 4
      for (int s = sl; s < a.nsplit; s += n)
        acc += *reinterpret_cast<const caf4*>(a.part + (s * stride + row) * a.dh + 4 * c) * fast_exp2(s_lse[s] - base);
    }
    s_acc[threadIdx.x] = acc;
    __syncthreads();
    const int unit = (int)(row / all), r = (int)(row - (int64_t)unit * all);
    int qi, hg;
    ca_row(a, r, qi, hg);
    const int64_t b = unit / a.Hk;
    const int h = (unit - (int)b * a.Hk) * a.G + hg;
    if (sl == 0 && 4 * c < a.dh) {
      for (int i = 1; i < n; ++i) acc += s_acc[i * tc + c];
      ca_store_out<DT>(a, ((b * a.Lq + qi) * a.Hk * a.G + h) * (int64_t)a.dh + 4 * c, acc * inv);
    }
    if (threadIdx.x == 0 && a.lse)
      a.lse[(b * a.Hk * a.G + h) * a.Lq + qi] = sum > 0.f ? (base + __log2f(sum)) * HCLSM_LN2 : sum != sum ? sum : -INFINITY;
    __syncthreads();
  }
}

// The same with one thread per four columns of a row, for many rows of few splits.
template <int DT>
__global__ void __launch_bounds__(256) ca_join_rows_kernel(const CaArgs a) {
  const int all = a.Lq * a.G;
  const uint32_t c4 = (uint32_t)a.dh / 4;
  const int64_t rows = (int64_t)a.units * all;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * c4; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / c4;
    const int col = (int)(i - row * c4) * 4;
    float top = -INFINITY, sum = 0.f;
    for (int s = 0; s < a.nsplit; ++s) top = fmaxf(top, a.part_lse[s * rows + row]);
    const float base = top == -INFINITY ? 0.f : top;
    caf4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < a.nsplit; ++s) {
      const float f = fast_exp2(a.part_lse[s * rows + row] - base);
      sum += f;
      acc += *reinterpret_cast<const caf4*>(a.part + (s * rows + row) * a.dh + col) * f;
    }
    const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    const int unit = (int)(row / all), r = (int)(row - (int64_t)unit * all);
    int qi, hg;
    ca_row(a, r, qi, hg);
    const int64_t b = unit / a.Hk;
    const int h = (unit - (int)b * a.Hk) * a.G + hg;
    ca_store_out<DT>(a, ((b * a.Lq + qi) * a.Hk * a.G + h) * (int64_t)a.dh + col, acc * inv);
    if (col == 0 && a.lse)
      a.lse[(b * a.Hk * a.G + h) * a.Lq + qi] = sum > 0.f ? (base + __log2f(sum)) * HCLSM_LN2 : sum != sum ? sum : -INFINITY;
  }
}

int ca_join(const CaArgs& a, int dtype, hipStream_t st) {
  if (a.nsplit <= 8) {
    const int64_t n = (int64_t)a.units * a.Lq * a.G * (a.dh / 4);
    const unsigned grid = (unsigned)((n + 255) / 256 < 8192 ? (n + 255) / 256 : 8192);
    if (dtype == HCLSM_F32) hipLaunchKernelGGL(ca_join_rows_kernel<HCLSM_F32>, dim3(grid), dim3(256), 0, st, a);
    else if (dtype == HCLSM_BF16) hipLaunchKernelGGL(ca_join_rows_kernel<HCLSM_BF16>, dim3(grid), dim3(256), 0, st, a);
    else hipLaunchKernelGGL(ca_join_rows_kernel<HCLSM_F16>, dim3(grid), dim3(256), 0, st, a);
    HCLSM_LAUNCH_CHECK();
    return 0;
  }
  const int64_t rows = (int64_t)a.units * a.Lq * a.G;
  int tc = 2;
  while (4 * tc < a.dh) tc *= 2;
  const unsigned grid = (unsigned)(rows < 65536 ? rows : 65536);
  if (dtype == HCLSM_F32) hipLaunchKernelGGL(ca_join_kernel<HCLSM_F32>, dim3(grid), dim3(256), 0, st, a, tc);
  else if (dtype == HCLSM_BF16) hipLaunchKernelGGL(ca_join_kernel<HCLSM_BF16>, dim3(grid), dim3(256), 0, st, a, tc);
  else hipLaunchKernelGGL(ca_join_kernel<HCLSM_F16>, dim3(grid), dim3(256), 0, st, a, tc);
  HCLSM_LAUNCH_CHECK();
  return 0;
}

// Partial sums of a split backward added in the splits' order, four columns to a thread.
template <int DT>
__global__ void __launch_bounds__(256) ca_sum_kernel(const CaArgs a, int keys) {
  const int rows = keys ? a.Lk : a.Lq * a.G;
  const uint32_t c4 = (uint32_t)a.dh / 4;
  const int64_t n = (int64_t)a.units * rows * c4, half = n * 4 * a.nsplit;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n * (keys ? 2 : 1); i += (int64_t)gridDim.x * 256) {
    const bool second = i >= n;
    const int64_t e = second ? i - n : i;
    const float* p = a.part + (second ? half : 0) + e * 4;
    caf4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int k = 0; k < a.nsplit; ++k) s += *reinterpret_cast<const caf4*>(p + (int64_t)k * n * 4);
    const int64_t row = e / c4;
    const int col = (int)(e - row * c4) * 4, unit = (int)(row / rows), r = (int)(row - (int64_t)unit * rows);
    const int64_t b = unit / a.Hk;
    const int hk = unit - (int)b * a.Hk;
    if (keys) {
      ca_store4<DT>(second ? a.dv : a.dk, ((b * a.Lk + r) * a.Hk + hk) * (int64_t)a.dh + col, s);
    } else {
      int qi, hg;
      ca_row(a, r, qi, hg);
      ca_store4<DT>(a.dq, ((b * a.Lq + qi) * a.Hk * a.G + hk * a.G + hg) * (int64_t)a.dh + col, s);
    }
  }
}

int ca_sum(const CaArgs& a, int keys, int dtype, hipStream_t st) {
  const int64_t n = (int64_t)a.units * (keys ? 2 * (int64_t)a.Lk : (int64_t)a.Lq * a.G) * (a.dh / 4);
  const unsigned grid = (unsigned)((n + 255) / 256 < 4096 ? (n + 255) / 256 : 4096);
  if (dtype == HCLSM_F32) hipLaunchKernelGGL(ca_sum_kernel<HCLSM_F32>, dim3(grid), dim3(256), 0, st, a, keys);
  else if (dtype == HCLSM_BF16) hipLaunchKernelGGL(ca_sum_kernel<HCLSM_BF16>, dim3(grid), dim3(256), 0, st, a, keys);
  else hipLaunchKernelGGL(ca_sum_kernel<HCLSM_F16>, dim3(grid), dim3(256), 0, st, a, keys);
  HCLSM_LAUNCH_CHECK();
  return 0;
}

namespace {

constexpr int64_t CA_MAX_DH = 256;

// Rows of 16 bytes' alignment: the kernels read and write whole 16-byte (outputs: 8-byte) vectors.
bool ca_aligned(const void* p, int64_t s0, int64_t s1, int64_t s2, int esz) {
  const int64_t n = 16 / esz;
  return (uintptr_t)p % 16 == 0 && s0 % n == 0 && s1 % n == 0 && s2 % n == 0;
}

// Partial sums are read and written as 16-byte vectors.
bool ca_workspace_aligned(const void* ws) { return (uintptr_t)ws % 16 == 0; }

// Offsets inside a tile (at most 64 rows, of a unit or of the keys) have to fit 31 bits.
bool ca_near(int64_t sl, int64_t sh, int64_t G, int esz) {
  return sl >= 0 && sh >= 0 && sl < (1 << 24) && sh < ((int64_t)1 << 31) && (64 / G + 2) * sl * esz + G * sh * esz < 0x7fff0000;
}

int ca_sizes(int64_t B, int64_t Lq, int64_t Lk, int64_t H, int64_t Hk, int64_t dh, int dtype) {
  if (B < 0 || Lq < 0 || Lk < 0 || H < 0 || Hk < 0 || dh < 1) return HCLSM_ERR_SHAPE;
  if (dtype < HCLSM_F32 || dtype > HCLSM_F16) return HCLSM_ERR_DTYPE;
  if (B > 0x7fffffff || Lq > 0x7fffffff || Lk > 0x7fffffff || H > 0x7fffffff) return HCLSM_ERR_SHAPE;
  if (H > 0 && (Hk == 0 || H % Hk != 0)) return HCLSM_ERR_SHAPE;
  if (dh > CA_MAX_DH || dh % 8 != 0) return HCLSM_ERR_UNSUPPORTED;
  // rows of a unit and units are int32; 128 to spare for tile arithmetic past the last row
  if (H > 0 && Lq > (0x7fffffff - 512) / (H / Hk)) return HCLSM_ERR_UNSUPPORTED;
  if (Lk > 0x7fffffff - 512) return HCLSM_ERR_UNSUPPORTED;
  if (Hk > 0 && B > (0x7fffffff - 8) / Hk) return HCLSM_ERR_UNSUPPORTED;
  return 0;
}

int ca_args(const HclsmCrossAttention* x, int bwd, CaArgs& a) {
  if (x == nullptr) return HCLSM_ERR_NULL;
  if (int rc = ca_sizes(x->B, x->Lq, x->Lk, x->H, x->Hk, x->dh, x->dtype)) return rc;
  if (!(x->scale > 0.f) || !(x->scale <= 2.0e38f)) return HCLSM_ERR_SHAPE;      // times log2(e) it is still finite
  const bool rows = x->B && x->Lq && x->H, keys = x->B && x->Lk && x->Hk;
  const int esz = x->dtype == HCLSM_F32 ? 4 : 2;
  const int64_t G = x->H ? x->H / x->Hk : 1;
  if (rows) {
    if (!ca_near(x->q_sl, x->q_sh, G, esz) || (bwd && !ca_near(x->g_sl, x->g_sh, G, esz))) return HCLSM_ERR_UNSUPPORTED;
    if (!x->q || !x->out || (bwd && (!x->g || !x->lse))) return HCLSM_ERR_NULL;
    if (!ca_aligned(x->q, x->q_sb, x->q_sl, x->q_sh, esz) || !ca_aligned(x->out, 0, 0, 0, esz) ||
        !ca_aligned(x->out_lo, 0, 0, 0, esz)) return HCLSM_ERR_UNSUPPORTED;
    if (bwd && (!ca_aligned(x->g, x->g_sb, x->g_sl, x->g_sh, esz) || !ca_aligned(x->dq, 0, 0, 0, esz)))
      return HCLSM_ERR_UNSUPPORTED;
  }
  if (keys) {
    if (!ca_near(x->k_sl, 0, 1, esz) || !ca_near(x->v_sl, 0, 1, esz)) return HCLSM_ERR_UNSUPPORTED;
    if (!x->k || !x->v || (bwd && (!x->dk != !x->dv))) return HCLSM_ERR_NULL;
    if (!ca_aligned(x->k, x->k_sb, x->k_sl, x->k_sh, esz) || !ca_aligned(x->v, x->v_sb, x->v_sl, x->v_sh, esz))
      return HCLSM_ERR_UNSUPPORTED;
    if (bwd && (!ca_aligned(x->dk, 0, 0, 0, esz) || !ca_aligned(x->dv, 0, 0, 0, esz))) return HCLSM_ERR_UNSUPPORTED;
  }
  for (int code : {x->key_lens_dtype, x->query_lens_dtype})
    if (code != HCLSM_POS_I32 && code != HCLSM_POS_I64) return HCLSM_ERR_DTYPE;
  a.q = (const char*)x->q; a.k = (const char*)x->k; a.v = (const char*)x->v; a.g = (const char*)x->g;
  a.o = (char*)x->out; a.olo = (char*)x->out_lo; a.dq = (char*)x->dq; a.dk = (char*)x->dk; a.dv = (char*)x->dv;
  a.lse = x->lse;
  a.qsb = x->q_sb; a.qsl = x->q_sl; a.qsh = x->q_sh;
  a.ksb = x->k_sb; a.ksl = x->k_sl; a.ksh = x->k_sh;
  a.vsb = x->v_sb; a.vsl = x->v_sl; a.vsh = x->v_sh;
  a.gsb = x->g_sb; a.gsl = x->g_sl; a.gsh = x->g_sh;
  a.pad = x->key_pad;
  a.psb = x->key_pad_sb;
  a.klens = x->key_lens; a.qlens = x->query_lens;
  a.klens64 = x->key_lens_dtype == HCLSM_POS_I64; a.qlens64 = x->query_lens_dtype == HCLSM_POS_I64;
  a.Hk = (int)x->Hk;
  a.G = x->H ? (int)(x->H / x->Hk) : 1;
  a.Lq = x->H ? (int)x->Lq : 0;        // no query head: no rows, whatever their length
  a.Lk = (int)x->Lk; a.dh = (int)x->dh;
  // row / G by a product: with 2^(l-1) < G <= 2^l and m = floor(2^(31+l) / G) + 1, floor(row m / 2^(31+l)) is
  // exact for row < 2^31
  a.gmul = 0;
  a.gshift = 0;
  if (a.G > 1) {
    int l = 1;
    while ((1ll << l) < a.G) ++l;
    a.gmul = (uint32_t)((1ull << (31 + l)) / (uint64_t)a.G + 1);
    a.gshift = l - 1;
  }
  a.scale = x->scale;
  a.scale_log2 = x->scale * HCLSM_LOG2E;
  return 0;
}

}  // namespace
}  // namespace hclsm

extern "C" int64_t hclsm_cross_attention_workspace(int64_t B, int64_t Lq, int64_t Lk, int64_t H, int64_t Hk, int64_t dh,
                                                   int dtype, int backward) {
  using namespace hclsm;
  if (int rc = ca_sizes(B, Lq, Lk, H, Hk, dh, dtype)) return rc;
  if (B == 0 || Hk == 0) return 0;
  if (backward) return ca_backward_bytes(ca_backward_plan(B, Lq, Lk, Hk, H / Hk, dh, dtype), B, Lq, Lk, Hk, H / Hk, dh);
  if (Lq == 0 || H == 0) return 0;
  const CaPlan p = ca_forward_plan(B, Lq, Lk, Hk, H / Hk, dh, dtype);
  return p.nsplit > 1 ? p.nsplit * B * Lq * H * (dh + 1) * 4 : 0;
}

extern "C" int hclsm_cross_attention_forward(const HclsmCrossAttention* x, void* workspace, int64_t workspace_bytes,
                                             void* stream) {
  using namespace hclsm;
  CaArgs a{};
  if (int rc = ca_args(x, 0, a)) return rc;
  if (x->B == 0 || x->Lq == 0 || x->H == 0) return 0;
  if (!ca_workspace_aligned(workspace)) return HCLSM_ERR_UNSUPPORTED;
  const hipStream_t st = (hipStream_t)stream;
  if (x->dtype == HCLSM_F32) return ca_forward_f32(a, x->B, workspace, workspace_bytes, st);
  if (x->dtype == HCLSM_BF16) return ca_forward_bf16(a, x->B, workspace, workspace_bytes, st);
  return ca_forward_f16(a, x->B, workspace, workspace_bytes, st);
}

extern "C" int hclsm_cross_attention_backward(const HclsmCrossAttention* x, void* workspace, int64_t workspace_bytes,
                                              void* stream) {
  using namespace hclsm;
  CaArgs a{};
  if (int rc = ca_args(x, 1, a)) return rc;
  if (x->B == 0 || x->Hk == 0 || (!x->dq && !x->dk)) return 0;
  const int64_t need = hclsm_cross_attention_workspace(x->B, x->Lq, x->Lk, x->H, x->Hk, x->dh, x->dtype, 1);
  if (need > 0 && workspace == nullptr) return HCLSM_ERR_NULL;
  if (workspace_bytes < need) return HCLSM_ERR_SHAPE;
  if (!ca_workspace_aligned(workspace)) return HCLSM_ERR_UNSUPPORTED;
  const hipStream_t st = (hipStream_t)stream;
  if (x->dtype == HCLSM_F32) return ca_backward_f32(a, x->B, workspace, workspace_bytes, st);
  if (x->dtype == HCLSM_BF16) return ca_backward_bf16(a, x->B, workspace, workspace_bytes, st);
  return ca_backward_f16(a, x->B, workspace, workspace_bytes, st);
}
