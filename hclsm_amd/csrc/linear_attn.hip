// Linear attention: argument checks, how a call is split, sums over segments and shared heads, and the form for one token.
#include "linear_attn.h"

namespace hclsm {

namespace {

// Segments of a call: where heads and columns alone are fewer workgroups than the chip has CUs, the tokens are split, each segment's
// sum formed first (from zero), the states in front of the segments from those, and then all segments at once: two workgroups to a
// CU, and four chunks or more to a segment.  The sums read B and X once more.  Measured (us):
//   50176 tokens, 12 heads of 64, bf16: 21 segments 140, 32: 130, 42 (the rule's): 116, 53: 124, 64: 119
//   2048 tokens in 1, 2, 3 and 4 segments, the rule's in brackets, by workgroups (64: eight segments)
//                      64                128              160               192               224               256
//     bf16 of 64      64 54 40 35 (34)   63 56 50 44 (44)  64 64 52 53 (50)  65 65 60 57 (64)  65 66 62 70 (64)  66 69 70 85 (64)
//     bf16 of 128     80 66 50 43 (47)   79 68 64 58 (56)  79 85 67 77 (65)  80 85 88 82 (85)  81 86 90 97 (85)  82 93 101 104 (82)
//     float16 of 64   98 80 58 48 (43)   98 82 74 61 (61)  99 102 76 88 (74) 101 102 100 89 (100) 102 102 104 102 (101) 103 105 108 109 (103)
//     float32 of 64   145 119 88 68 (56) 147 123 110 93 (89) 147 152 117 118 (113) 149 155 135 130 (159) 150 163 149 165 (162) 155 174 165 179 (159)
//   one prompt, 12 heads of 64, unsplit, in segments of two chunks (the rule's): bf16 128 tokens 8.1 11.1 (8.1), 256: 11.6 13.6
//     (11.6), 512: 19.0 14.8 (18.7), 1024: 33.2 18.1 (20.1); float32 128: 12.6 12.7 (12.7), 256: 21.5 15.9 (21.3), 512: 38.5 19.3 (22.8)
// So two segments of 171 to 255 workgroups take 5% less to 8% more, where four would take up to 13% less below 200 for heads of 64, and
// segments of two chunks would gain a fifth for short prompts of six chunks or more.
struct LaPlan {
  int nseg, seg_tokens;
};

LaPlan la_plan(int64_t workgroups, int64_t L, int chunk) {
  const int64_t chunks = (L + chunk - 1) / chunk;
  int64_t n = workgroups > 0 ? (workgroups < 256 ? 512 / workgroups : 1) : 1;
  n = n > chunks / 4 ? chunks / 4 : n;
  n = n > LA_MAX_SEGMENTS ? LA_MAX_SEGMENTS : n;
  if (n <= 1) return {1, 0};
  const int64_t per = (chunks + n - 1) / n;
  return {(int)((chunks + per - 1) / per), (int)(per * chunk)};
}

int64_t la_up(int64_t n) { return (n + 255) / 256 * 256; }

struct LaSizes {
  int64_t B, L, H, Hk, dk, dv;
  int dtype;
  int64_t units() const { return B * H; }
  int64_t tiles(int64_t dx) const { return (dx + LA_XT - 1) / LA_XT; }
  // chunks of the widest job decide for all jobs of a call
  int chunk(bool bwd) const {
    const int c = la_chunk(dtype, la_padded(dk)), d = la_chunk(dtype, la_padded(dv));
    return bwd && d > c ? d : c;
  }
  int64_t column_tiles(bool bwd) const { return bwd ? tiles(dv) + 2 * tiles(dk) : tiles(dv); }      // of all jobs
  LaPlan plan(bool bwd) const { return la_plan(units() * column_tiles(bwd), L, chunk(bwd)); }
  int64_t seg_bytes(bool bwd) const {
    const LaPlan p = plan(bwd);
    return p.nseg > 1 ? la_up(units() * p.nseg * dk * dv * 4) : 0;
  }
  int64_t workspace(bool bwd) const {
    if (!bwd) return seg_bytes(false);
    return 3 * seg_bytes(true) + (H > Hk ? la_up(B * L * H * dk * 4) + la_up(B * L * H * dv * 4) : 0);
  }
};

int la_sizes(const LaSizes& z) {
  if (z.B < 0 || z.L < 0 || z.H < 0 || z.Hk < 0 || z.dk < 1 || z.dv < 1) return HCLSM_ERR_SHAPE;
  if (z.dtype < HCLSM_F32 || z.dtype > HCLSM_F16) return HCLSM_ERR_DTYPE;
  if (z.H > 0 && (z.Hk == 0 || z.H % z.Hk != 0)) return HCLSM_ERR_SHAPE;
  if (z.dk > LA_MAX_DIM || z.dv > LA_MAX_DIM || z.dk % 8 || z.dv % 8) return HCLSM_ERR_UNSUPPORTED;
  // workgroups of one launch (three jobs of up to four column tiles) have fewer than 2^32 threads
  if (z.B > 0x7fffffff || z.H > 0x7fffffff || z.L > 0x7fffffff - 1024) return HCLSM_ERR_UNSUPPORTED;
  if (z.H > 0 && z.B > (1 << 20) / z.H) return HCLSM_ERR_UNSUPPORTED;
  // a chunk's outputs lie within 31 bits of each other
  if (z.H * (z.dk > z.dv ? z.dk : z.dv) >= 1 << 23) return HCLSM_ERR_UNSUPPORTED;
  return 0;
}

// and so do its inputs (chunks of float32 have 32 tokens)
bool la_near(int64_t sl) { return sl >= 0 && sl < 1 << 23; }

bool la_aligned(const void* p, int64_t s0, int64_t s1, int64_t s2, int esz) {
  const int64_t n = 16 / esz;
  return (uintptr_t)p % 16 == 0 && s0 % n == 0 && s1 % n == 0 && s2 % n == 0;
}

// States in front of a call's segments, from the sums of the segments before them, in place.  One thread per element: the segments
// one after another, the loads of 16 in flight.  Latency bounds it: 10 us for 42 segments of 12 heads of 64 x 64 (8.3 MB read
// and written).  Groups of segments by threads of their own, joined through LDS, took 24 us where this took 11.5, 32 loads no less.
__global__ void __launch_bounds__(256) la_prefix_kernel(const LaArgs a) {
  const LaJob& j = a.job[blockIdx.y];
  const int n = j.da * j.dx, blocks = (n + 255) / 256, unit = (int)blockIdx.x / blocks, b = unit / a.H, h = unit - b * a.H;
  const int e = ((int)blockIdx.x - unit * blocks) * 256 + threadIdx.x;
  if (e >= n) return;
  const int live = ca_len(a.lens, a.lens64, b, a.L);
  const float g = la_log_decay(a.log_decay, h);
  const int d = e / j.dx, c = e - d * j.dx;
  float* p = j.seg + (int64_t)unit * a.nseg * n + e;
  float s = j.s0 ? j.s0[(int64_t)unit * n + d * j.s_r + c * j.s_c] : 0.f;
  int64_t of = a.seg_tokens;      // tokens that `an` and `less` are for
  float an = expf(g * (float)of), less = expm1f(g * (float)of);
  constexpr int NB = 16;
  for (int k0 = 0; k0 < a.nseg; k0 += NB) {
    float u[NB];
#pragma unroll
    for (int k = 0; k < NB; ++k) u[k] = k0 + k + 1 < a.nseg ? p[(int64_t)(k0 + k) * n] : 0.f;
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      if (k0 + k >= a.nseg) break;
      const int64_t t0 = (int64_t)(j.back ? a.nseg - 1 - k0 - k : k0 + k) * a.seg_tokens;
      const int64_t m = live - t0 < 0 ? 0 : live - t0 > a.seg_tokens ? a.seg_tokens : live - t0;
      p[(int64_t)(k0 + k) * n] = s;
      if (m != of) {
        of = m;
        an = expf(g * (float)m);
        less = expm1f(g * (float)m);
      }
      s = la_decayed(s, an, less) + u[k];
    }
  }
}

// Gradients of shared heads: the sums of the heads of a group, rounded once, in the heads' order.  One pass over the heads' float32
// gradients (HBM); adding them in the main kernel would need the heads of a group in one workgroup, or atomics.
template <int DT> __global__ void __launch_bounds__(256) la_group_kernel(const float* ws, char* y, int64_t n, int G, int d4) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / d4, c = i - row * d4;
    caf4 s = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < G; ++k) s += *reinterpret_cast<const caf4*>(ws + ((row * G + k) * d4 + c) * 4);
    ca_store4<DT>(y, i * 4, s);
  }
}

int la_group(const float* ws, void* y, int64_t rows, int G, int64_t d, int dtype, hipStream_t st) {
  const int64_t n = rows * (d / 4);
  if (n == 0) return 0;
  const dim3 grid((unsigned)((n + 255) / 256 < 8192 ? (n + 255) / 256 : 8192));
  if (dtype == HCLSM_F32) hipLaunchKernelGGL(la_group_kernel<HCLSM_F32>, grid, dim3(256), 0, st, ws, (char*)y, n, G, (int)(d / 4));
  else if (dtype == HCLSM_BF16) hipLaunchKernelGGL(la_group_kernel<HCLSM_BF16>, grid, dim3(256), 0, st, ws, (char*)y, n, G, (int)(d / 4));
  else hipLaunchKernelGGL(la_group_kernel<HCLSM_F16>, grid, dim3(256), 0, st, ws, (char*)y, n, G, (int)(d / 4));
  HCLSM_LAUNCH_CHECK();
  return 0;
}

int la_launch_any(const LaArgs& a, int dtype, int da, bool sum, hipStream_t st) {
  if (dtype == HCLSM_F32) return la_launch_f32(a, da, sum, st);
  if (dtype == HCLSM_BF16) return la_launch_bf16(a, da, sum, st);
  return la_launch_f16(a, da, sum, st);
}

// All jobs of a call: sums of segments, states in front of them, outputs.  Jobs of the same padded sizes share a launch.
int la_run(LaArgs a, const LaSizes& z, bool bwd, hipStream_t st) {
  // Jobs of different padded sizes share a launch of the larger one where together they are on the chip at once (two workgroups
  // to each of 256 CUs): they then run side by side.  Elsewhere the padding would cost, and they run one after the other.  All
  // jobs that the sizes have count, wanted or not: a job's chunks, and so its bits, follow from its padded size.
  const int64_t all = z.units() * a.nseg * z.column_tiles(bwd);
  const int64_t most = bwd && z.dv > z.dk ? z.dv : z.dk;
  auto padded = [&](int i) { return la_padded(all <= 512 ? most : a.job[i].da); };
  for (int pass = a.nseg > 1 ? 0 : 2; pass < 3; ++pass) {
    if (pass == 1) {
      if (a.nseg <= LA_FEW_SEGMENTS) continue;      // the main kernel adds them up itself
      const int64_t n = ((int64_t)a.job[0].da * a.job[0].dx + 255) / 256 * a.B * a.H;
      hipLaunchKernelGGL(la_prefix_kernel, dim3((unsigned)n, (unsigned)a.njobs), dim3(256), 0, st, a);
      HCLSM_LAUNCH_CHECK();
      continue;
    }
    bool done[3] = {false, false, false};
    for (int i = 0; i < a.njobs; ++i) {
      if (done[i]) continue;
      LaArgs one = a;
      one.njobs = 0;
      one.per = 0;
      const int da = padded(i);
      for (int k = i; k < a.njobs; ++k) {
        if (done[k] || padded(k) != da) continue;
        done[k] = true;
        one.per += (uint32_t)a.job[k].xtiles;
        one.job[one.njobs++] = a.job[k];
      }
      one.items = a.B * a.H * a.nseg;
      one.by_xcd = one.items >= 64;
      if (int rc = la_launch_any(one, z.dtype, da, pass == 0, st)) return rc;
    }
  }
  return 0;
}

int la_args(const HclsmLinearAttention* x, bool bwd, LaSizes& z) {
  if (x == nullptr) return HCLSM_ERR_NULL;
  z = LaSizes{x->B, x->L, x->H, x->Hk, x->dk, x->dv, x->dtype};
  if (int rc = la_sizes(z)) return rc;
  if (!(x->scale > 0.f) || !(x->scale <= 3.0e38f)) return HCLSM_ERR_SHAPE;
  if (x->seq_lens_dtype != HCLSM_POS_I32 && x->seq_lens_dtype != HCLSM_POS_I64) return HCLSM_ERR_DTYPE;
  if (z.B == 0 || z.H == 0) return 0;
  const int esz = z.dtype == HCLSM_F32 ? 4 : 2;
  if (x->log_decay == nullptr) return HCLSM_ERR_NULL;
  if (z.L > 0) {
    if (!x->q || !x->k || !x->v || (bwd ? !x->g : !x->out)) return HCLSM_ERR_NULL;
    if (!la_aligned(x->q, x->q_sb, x->q_sl, x->q_sh, esz) || !la_aligned(x->k, x->k_sb, x->k_sl, x->k_sh, esz) ||
        !la_aligned(x->v, x->v_sb, x->v_sl, x->v_sh, esz)) return HCLSM_ERR_UNSUPPORTED;
    if (!la_near(x->q_sl) || !la_near(x->k_sl) || !la_near(x->v_sl) || (bwd && !la_near(x->g_sl))) return HCLSM_ERR_UNSUPPORTED;
    if (bwd ? !la_aligned(x->g, x->g_sb, x->g_sl, x->g_sh, esz) : !la_aligned(x->out, 0, 0, 0, esz)) return HCLSM_ERR_UNSUPPORTED;
    if (bwd && (!la_aligned(x->dq, 0, 0, 0, esz) || !la_aligned(x->dk_out, 0, 0, 0, esz) || !la_aligned(x->dv_out, 0, 0, 0, esz)))
      return HCLSM_ERR_UNSUPPORTED;
  }
  return 0;
}

LaTensor la_tensor(const void* p, int64_t sb, int64_t sl, int64_t sh, int64_t group) {
  return {(const char*)p, sb, sl, sh, (int)group};
}

LaArgs la_common(const HclsmLinearAttention* x, const LaPlan& p) {
  LaArgs a{};
  a.log_decay = x->log_decay;
  a.lens = x->seq_lens;
  a.lens64 = x->seq_lens_dtype == HCLSM_POS_I64;
  a.B = (int)x->B; a.H = (int)x->H; a.L = (int)x->L;
  a.nseg = p.nseg;
  a.seg_tokens = p.seg_tokens;
  return a;
}

}  // namespace

// One token: S = a S + k v^T in place, o = c q^T S.  A workgroup has 64 columns of one head's state: 16 lanes of four columns,
// 16 groups of rows.  Each state is read and written once, which bounds it (HBM); the loads of eight rows are in flight: 111 us for
// 256 states of 16 heads of 128 x 128 (537 MB, 4.9 TB/s, a copy's rate), 5.0 for 16 of 12 heads of 64 x 64 (latency).
constexpr int LS_COLS = 64, LS_GROUPS = 16, LS_BATCH = 8;

struct LsArgs {
  const void *q, *k, *v;
  int64_t qsb, qsh, ksb, ksh, vsb, vsh, ssb;
  const float* log_decay;
  float* s;
  const void* rows;
  int64_t n_states;
  char* out;
  int rows64, H, G, dk, dv, tiles;
  float scale;
};

template <int DT> __global__ void __launch_bounds__(256) la_step_kernel(const LsArgs a) {
  using E = typename Elem<DT>::T;
  __shared__ float sq[LA_MAX_DIM], sk[LA_MAX_DIM];
  __shared__ caf4 part[4][16];
  const uint32_t u = blockIdx.x / (uint32_t)a.tiles, tile = blockIdx.x - u * (uint32_t)a.tiles;
  const uint32_t b = u / (uint32_t)a.H, h = u - b * (uint32_t)a.H;
  const int hk = (int)h / a.G, lane = threadIdx.x & 15, grp = threadIdx.x >> 4;
  const int col = (int)tile * LS_COLS + 4 * lane;
  int64_t row = b;
  if (a.rows) row = a.rows64 ? reinterpret_cast<const int64_t*>(a.rows)[b] : (int64_t)reinterpret_cast<const int32_t*>(a.rows)[b];
  const bool in = row >= 0 && row < a.n_states;
  caf4 acc = {0.f, 0.f, 0.f, 0.f};
  if (in) {
    float* s = a.s + row * a.ssb + (int64_t)h * a.dk * a.dv + col;
    const bool mine = col < a.dv;
    caf4 t[LS_BATCH];
    auto load = [&](int d0) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < LS_BATCH; ++i) {
        const int d = d0 + grp + i * LS_GROUPS;
        if (mine && d < a.dk) t[i] = *reinterpret_cast<const caf4*>(s + (int64_t)d * a.dv);
      }
    };
    load(0);
    for (int d = threadIdx.x; d < a.dk; d += 256) {
      sq[d] = Elem<DT>::ld(reinterpret_cast<const E*>(a.q) + b * a.qsb + h * a.qsh + d) * a.scale;
      sk[d] = Elem<DT>::ld(reinterpret_cast<const E*>(a.k) + b * a.ksb + hk * a.ksh + d);
    }
    caf4 v = {0.f, 0.f, 0.f, 0.f};
    if (mine) {
      const E* p = reinterpret_cast<const E*>(a.v) + b * a.vsb + hk * a.vsh + col;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = Elem<DT>::ld(p + i);
    }
    // a S + k v^T: near one as S + ((a - 1) S + k v^T), rounded once at the size of the state, and by tokens independently of
    // each other; a rounded a would be off alike for every token (at -2^-12, after 4096 tokens, by 1076 x 2^-24 of the state, as it is by 17)
    const float gd = la_log_decay(a.log_decay, (int)h), an = expf(gd);
    const bool slow = an >= 0.5f;
    const float decay = slow ? expm1f(gd) : an;
    __syncthreads();
    for (int d0 = 0; d0 < a.dk; d0 += LS_BATCH * LS_GROUPS) {
#pragma unroll
      for (int i = 0; i < LS_BATCH; ++i) {
        const int d = d0 + grp + i * LS_GROUPS;
        if (mine && d < a.dk) {
          const float q = sq[d], k = sk[d];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float add = fmaf(t[i][e], decay, k * v[e]);
            t[i][e] = slow ? t[i][e] + add : add;
            acc[e] = fmaf(q, t[i][e], acc[e]);
          }
          *reinterpret_cast<caf4*>(s + (int64_t)d * a.dv) = t[i];
        }
      }
      if (d0 + LS_BATCH * LS_GROUPS < a.dk) load(d0 + LS_BATCH * LS_GROUPS);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = rows4_sum(acc[e]);
    if ((threadIdx.x & 63) < 16) part[threadIdx.x >> 6][lane] = acc;
    __syncthreads();
    acc = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
  }
  if (threadIdx.x < 16 && col < a.dv) ca_store4<DT>(a.out, (int64_t)u * a.dv + col, acc);
}

}  // namespace hclsm

extern "C" int64_t hclsm_linear_attention_workspace(int64_t B, int64_t L, int64_t H, int64_t Hk, int64_t dk, int64_t dv,
                                                    int dtype, int backward) {
  using namespace hclsm;
  const LaSizes z{B, L, H, Hk, dk, dv, dtype};
  if (int rc = la_sizes(z)) return rc;
  if (B == 0 || H == 0) return 0;
  return z.workspace(backward != 0);
}

extern "C" int hclsm_linear_attention_forward(const HclsmLinearAttention* x, void* workspace, int64_t workspace_bytes,
                                              void* stream) {
  using namespace hclsm;
  LaSizes z;
  if (int rc = la_args(x, false, z)) return rc;
  if (z.B == 0 || z.H == 0 || (z.L == 0 && x->state_out == nullptr)) return 0;
  const int64_t need = z.workspace(false);
  if (need > 0 && workspace == nullptr) return HCLSM_ERR_NULL;
  if (workspace_bytes < need) return HCLSM_ERR_SHAPE;
  if ((uintptr_t)workspace % 16) return HCLSM_ERR_UNSUPPORTED;
  const int64_t G = z.H / z.Hk;
  LaArgs a = la_common(x, z.plan(false));
  a.njobs = 1;
  LaJob& o = a.job[0];
  o.a = la_tensor(x->q, x->q_sb, x->q_sl, x->q_sh, 1);
  o.b = la_tensor(x->k, x->k_sb, x->k_sl, x->k_sh, G);
  o.x = la_tensor(x->v, x->v_sb, x->v_sl, x->v_sh, G);
  o.y = (char*)x->out;
  o.s0 = x->state_in;
  o.s1 = x->state_out;
  o.seg = (float*)workspace;
  o.s_r = (int)z.dv;
  o.s_c = 1;
  a.fine = x->state_out != nullptr;
  o.da = (int)z.dk; o.dx = (int)z.dv;
  o.xtiles = (int)z.tiles(z.dv);
  o.cp = o.ci = x->scale;
  o.cu = 1.f;
  return la_run(a, z, false, (hipStream_t)stream);
}

extern "C" int hclsm_linear_attention_backward(const HclsmLinearAttention* x, void* workspace, int64_t workspace_bytes,
                                               void* stream) {
  using namespace hclsm;
  LaSizes z;
  if (int rc = la_args(x, true, z)) return rc;
  if (z.B == 0 || z.H == 0) return 0;
  const int64_t need = z.workspace(true);
  if (need > 0 && workspace == nullptr) return HCLSM_ERR_NULL;
  if (workspace_bytes < need) return HCLSM_ERR_SHAPE;
  if ((uintptr_t)workspace % 16) return HCLSM_ERR_UNSUPPORTED;
  const hipStream_t st = (hipStream_t)stream;
  const int64_t G = z.H / z.Hk, seg = z.seg_bytes(true);
  char* ws = (char*)workspace;
  float* wk = (float*)(ws + 3 * seg);
  float* wv = (float*)(ws + 3 * seg + la_up(z.B * z.L * z.H * z.dk * 4));
  LaArgs a = la_common(x, z.plan(true));
  a.fine = x->dstate_in || x->state_in;      // whether its gradient is wanted or not: the others have the same bits
  const LaTensor q = la_tensor(x->q, x->q_sb, x->q_sl, x->q_sh, 1), k = la_tensor(x->k, x->k_sb, x->k_sl, x->k_sh, G),
                 v = la_tensor(x->v, x->v_sb, x->v_sl, x->v_sh, G), g = la_tensor(x->g, x->g_sb, x->g_sl, x->g_sh, 1);
  auto job = [&](const LaTensor& ta, const LaTensor& tb, const LaTensor& tx, int64_t da, int64_t dx, bool turned) {
    LaJob& j = a.job[a.njobs];
    j.a = ta; j.b = tb; j.x = tx;
    j.da = (int)da; j.dx = (int)dx;
    j.xtiles = (int)z.tiles(dx);
    j.s_r = turned ? 1 : (int)z.dv;
    j.s_c = turned ? (int)z.dv : 1;
    j.seg = (float*)(ws + a.njobs * seg);
    j.cp = x->scale;
    ++a.njobs;
    return &j;
  };
  if (x->dq) {
    LaJob* j = job(g, v, k, z.dv, z.dk, true);
    j->y = (char*)x->dq;
    j->s0 = x->state_in;
    j->ci = x->scale;
    j->cu = 1.f;
  }
  if (x->dv_out || x->dstate_in) {
    LaJob* j = job(k, q, g, z.dk, z.dv, false);
    j->y = x->dv_out ? (G > 1 ? (char*)wv : (char*)x->dv_out) : nullptr;
    j->y32 = G > 1;
    j->s0 = x->dstate_out;
    j->s1 = x->dstate_in;
    j->ci = 1.f;
    j->cu = x->scale;
    j->shift = 1;
    j->back = 1;
  }
  if (x->dk_out) {
    LaJob* j = job(v, g, q, z.dv, z.dk, true);
    j->y = G > 1 ? (char*)wk : (char*)x->dk_out;
    j->y32 = G > 1;
    j->s0 = x->dstate_out;
    j->ci = 1.f;
    j->cu = x->scale;
    j->shift = 1;
    j->back = 1;
  }
  if (a.njobs == 0) return 0;
  if (int rc = la_run(a, z, true, st)) return rc;
  if (G > 1 && x->dk_out)
    if (int rc = la_group(wk, x->dk_out, z.B * z.L * z.Hk, (int)G, z.dk, z.dtype, st)) return rc;
  if (G > 1 && x->dv_out)
    if (int rc = la_group(wv, x->dv_out, z.B * z.L * z.Hk, (int)G, z.dv, z.dtype, st)) return rc;
  return 0;
}

extern "C" int hclsm_linear_attention_step(const HclsmLinearAttentionStep* x, void* stream) {
  using namespace hclsm;
  if (x == nullptr) return HCLSM_ERR_NULL;
  if (int rc = la_sizes(LaSizes{x->B, 1, x->H, x->Hk, x->dk, x->dv, x->dtype})) return rc;
  if (!(x->scale > 0.f) || !(x->scale <= 3.0e38f) || x->n_states < 0) return HCLSM_ERR_SHAPE;
  if (x->rows_dtype != HCLSM_POS_I32 && x->rows_dtype != HCLSM_POS_I64) return HCLSM_ERR_DTYPE;
  if (x->B == 0 || x->H == 0) return 0;
  if (!x->rows && x->n_states < x->B) return HCLSM_ERR_SHAPE;
  if (!x->q || !x->k || !x->v || !x->log_decay || !x->out || (!x->state && x->n_states > 0)) return HCLSM_ERR_NULL;
  if ((uintptr_t)x->state % 16 || x->state_sb % 4 || (uintptr_t)x->out % 16) return HCLSM_ERR_UNSUPPORTED;
  LsArgs a{};
  a.q = x->q; a.k = x->k; a.v = x->v;
  a.qsb = x->q_sb; a.qsh = x->q_sh; a.ksb = x->k_sb; a.ksh = x->k_sh; a.vsb = x->v_sb; a.vsh = x->v_sh;
  a.ssb = x->state_sb;
  a.log_decay = x->log_decay;
  a.s = x->state;
  a.rows = x->rows;
  a.rows64 = x->rows_dtype == HCLSM_POS_I64;
  a.n_states = x->n_states;
  a.out = (char*)x->out;
  a.H = (int)x->H; a.G = (int)(x->H / x->Hk); a.dk = (int)x->dk; a.dv = (int)x->dv;
  a.tiles = (a.dv + LS_COLS - 1) / LS_COLS;
  a.scale = x->scale;
  const dim3 grid((unsigned)(x->B * x->H * a.tiles));
  const hipStream_t st = (hipStream_t)stream;
  if (x->dtype == HCLSM_F32) hipLaunchKernelGGL(la_step_kernel<HCLSM_F32>, grid, dim3(256), 0, st, a);
  else if (x->dtype == HCLSM_BF16) hipLaunchKernelGGL(la_step_kernel<HCLSM_BF16>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(la_step_kernel<HCLSM_F16>, grid, dim3(256), 0, st, a);
  HCLSM_LAUNCH_CHECK();
  return 0;
}
