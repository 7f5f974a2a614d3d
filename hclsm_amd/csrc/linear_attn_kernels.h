// The chunked kernel of linear attention, instantiated for one element type per source file (linear_attn_*.hip).
#pragma once

#include "cross_attn_stage.h"
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

// N planes of four and of eight float32 values.
template <int N> __device__ __forceinline__ void la_split(caf4 v, uint2* out) {
#pragma unroll
  for (int p = 0; p < N; ++p) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
      if (p + 1 < N) {
        asm("" : "+v"(w[i]));      // (the pair as it is: otherwise each element's conversion is repeated for its rest)
        v[2 * i] -= LaB::lo(w[i]);
        v[2 * i + 1] -= LaB::hi(w[i]);
      }
    }
    out[p] = uint2{w[0], w[1]};
  }
}
template <int N> __device__ __forceinline__ void la_split(const float* v, uint4* out) {
  uint2 a[N], b[N];
  la_split<N>(caf4{v[0], v[1], v[2], v[3]}, a);
  la_split<N>(caf4{v[4], v[5], v[6], v[7]}, b);
#pragma unroll
  for (int p = 0; p < N; ++p) out[p] = uint4{a[p].x, a[p].y, b[p].x, b[p].y};
}
template <int N> __device__ __forceinline__ void la_split(const caf4* t, LaFrag* out) {
  const float v[8] = {t[0][0], t[0][1], t[0][2], t[0][3], t[1][0], t[1][1], t[1][2], t[1][3]};
  uint4 w[N];
  la_split<N>(v, w);
#pragma unroll
  for (int p = 0; p < N; ++p) out[p] = ca_frag<HCLSM_BF16>(w[p]);
}

// Rows of one chunk on their way from global memory to LDS: row r of the tile is token r, or n - 1 - r backwards, of the chunk's n
// live ones; other rows and columns past d are zeros (a load past the buffer resource's end gives zeros).  bf16 goes straight
// to LDS, the other types through registers, in which they are split into their planes.  The offsets stand for a number of live
// tokens: they are formed again when that changes.
template <int DT, int C, int D, int NT> struct LaStage {
  static constexpr bool DMA = DT == HCLSM_BF16;
  static constexpr int U = C * (D / 8) / NT, RAW = LaT<DT>::RAW, NP = LaT<DT>::NP, ESZ = DT == HCLSM_F32 ? 4 : 2;
  using Tile = CaTile<HCLSM_BF16, D>;
  static_assert(Tile::PC == D / 8 && C * (D / 8) % NT == 0, "rows without padding, whole units");
  static constexpr int PLANE = C * Tile::STRIDE, BYTES = NP * PLANE;
  static constexpr uint32_t NONE = 0xffffffffu;
  static constexpr int STEP = NT / (D / 8);     // rows between a thread's units, which therefore have the same chunk
  static_assert(STEP % 8 == 0, "rows of a thread differ by multiples of 8");
  uint4 raw[DMA ? 1 : U][RAW];

  static __device__ __forceinline__ int row(int u) { return ((int)threadIdx.x + u * NT) / (D / 8); }
  static __device__ __forceinline__ int chunk(int u) { return (((int)threadIdx.x + u * NT) % (D / 8)) ^ Tile::swap(row(u)); }

  // base: the chunk's first token at column 0; sb: bytes between tokens; n live tokens, d columns
  __device__ __forceinline__ void load(const char* base, int sb, int n, int d, bool back, char* t, int wave) {
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 0x7fffffff, kRawBufferWord3);
    const int r0 = row(0), c0 = chunk(0) * 8;
    auto one = [&](int u, int off, int so) __attribute__((always_inline)) {
      if constexpr (DMA) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (ca_lds_void*)(t + (u * NT + wave * 64) * 16), 16, off, so, 0, 0);
      } else {
#pragma unroll
        for (int k = 0; k < RAW; ++k)
          raw[u][k] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rs, off, so + 16 * k, 0));
      }
    };
    if (n == C) {
      // row r0 + u STEP, backwards C - 1 - r0 - u STEP
      const int off = c0 < d ? (back ? C - 1 - (U - 1) * STEP - r0 : r0) * sb + c0 * ESZ : (int)NONE;
#pragma unroll
      for (int u = 0; u < U; ++u) one(u, off, __builtin_amdgcn_readfirstlane((back ? U - 1 - u : u) * STEP * sb));
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = r0 + u * STEP;
        one(u, r < n && c0 < d ? (back ? n - 1 - r : r) * sb + c0 * ESZ : (int)NONE, 0);
      }
    }
  }
  __device__ __forceinline__ void store(char* t) const {
    if constexpr (!DMA) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
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
        uint4 w[NP];
        la_split<NP>(v, w);
#pragma unroll
        for (int p = 0; p < NP; ++p) *reinterpret_cast<uint4*>(t + p * PLANE + ((int)threadIdx.x + u * NT) * 16) = w[p];
      }
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

// acc[t] += a b[t] for every t, over the planes whose orders add up to at most MOST (what is left out lies below the last plane
// kept): products in a row have results of their own.
template <int NA, int NB, int MOST, int T> __device__ __forceinline__ void la_mma_all(const LaFrag* a, const LaFrag (*b)[NB], caf4* acc) {
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
      if (i + j <= MOST)
#pragma unroll
        for (int t = 0; t < T; ++t) acc[t] = LaB::mma(a[i], b[t][j], acc[t]);
}
template <int NA, int NB, int MOST, int T> __device__ __forceinline__ void la_mma_all(const LaFrag (*a)[NA], const LaFrag* b, caf4* acc) {
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
      if (i + j <= MOST)
#pragma unroll
        for (int t = 0; t < T; ++t) acc[t] = LaB::mma(a[t][i], b[j], acc[t]);
}

// A barrier for what went through LDS: loads and transfers from global memory stay in flight (__syncthreads waits for them).
__device__ __forceinline__ void la_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);      // LDS counter zero (gfx9 encoding), the others as they are
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// S += B^T X for 32 tokens' weighted X (v, the lane's column and tokens) in N planes; two tiles of S at a time, the
// operands of the next two on their way (four: heads of 256 spill, 217 -> 245 us, float16 of 128 192 for 186).
template <int DA, int NP, int N, int PLANE>
__device__ __forceinline__ void la_update(char* tb, int row0, const float* v, caf4* s, int li, int g) {
  constexpr int M = DA / 16, T = 2;
  LaFrag fb[2][T][NP];
  auto get = [&](int m0, LaFrag (*f)[NP]) __attribute__((always_inline)) {
#pragma unroll
    for (int m = 0; m < T; ++m)
#pragma unroll
      for (int p = 0; p < NP; ++p) f[m][p] = la_frag_cols<DA>(tb + p * PLANE, row0, (m0 + m) >> 1, (m0 + m) & 1, li, g);
  };
  get(0, fb[0]);
  uint4 w[N];
  la_split<N>(v, w);
  LaFrag fw[N];
#pragma unroll
  for (int p = 0; p < N; ++p) fw[p] = ca_frag<HCLSM_BF16>(w[p]);
#pragma unroll
  for (int m = 0; m < M; m += T) {
    if (m + T < M) get(m + T, fb[(m / T + 1) & 1]);
    ca_fence();
    la_mma_all<NP, N, N - 1, T>(fb[m / T & 1], fw, s + m);
    ca_fence();
  }
}

// One workgroup of four waves: a head of a batch row, 64 columns of X (and of the state and the output), one segment of the
// tokens, chunk after chunk.  Wave w owns 16 columns of the state, in registers for the whole segment; the weights of
// pairs (A_r . B_s) a^(r-s) are shared out over the waves and passed through LDS in the order in which the matrix unit
// reads them.  Several workgroups of a CU hide each other's waits.  SUM: the state alone, from zero (the sum of a segment).
//
// Why 64 columns: A and B are read once for each column tile (from L2: the tiles of a head run on one XCD), and 64 leaves the
// registers and LDS for two or three workgroups to a CU; 128 columns by eight waves, one workgroup to a CU, took 996 us where
// 64 took 746 (8 x 4096 tokens, below).  Why 64 tokens: the state's share, 4 dk dv flops a token, does not depend on it, the pairs' grows with it,
// and the planes of the state are formed once for each chunk.  Why two buffers of B and X: with one of each the same call took
// 746 us, before they were 653; two chunks ahead in three buffers, where the LDS has the room (sums alone), gained nothing.
// What bounds it, bf16: heads of 64, HBM (32 x 1024 tokens, 12 heads, with gradients: 165 us, 704 MB, 4.3 TB/s; 50176 tokens of 12
// heads, split over time, main launch 73 us, 4.2 TB/s).  Heads of 128 (8 x 4096 tokens, 16 heads, with gradients: 555 to 585
// us, 3.3 TB/s): vector unit 40%, matrix unit 30%, LDS 31% of the backward's cycles, in turn, since two waves per SIMD do not cover
// each other's waits.  float16 takes 1.4 to 2.5 times and float32 2.1 to 3.8 times as long: two and three planes for each
// input, formed on the way to LDS.  (Each wait on the transfers in flight that the compiler adds shows: for writes to LDS that
// it joins, spills, stores that only some paths make.)
template <int DT, int DA, bool SUM>
__global__ void __launch_bounds__(LA_THREADS, la_waves(DT, DA)) la_kernel(const LaArgs args) {
  constexpr int NT = LA_THREADS, XT = LA_XT, C = la_chunk(DT, DA), KT = C / 16, NS = DA / 16, NP = LaT<DT>::NP,
                NC = LaT<DT>::NC;
  constexpr int ESZ = DT == HCLSM_F32 ? 4 : 2, MOST = NC - 1;
  constexpr int NF = KT == 4 ? 6 : 2;     // 16 tokens by 32 at or below the diagonal
  using SA = LaStage<DT, C, DA, NT>;
  using SX = LaStage<DT, C, XT, NT>;
  using TA = CaTile<HCLSM_BF16, DA>;
  using TX = CaTile<HCLSM_BF16, XT>;
  constexpr bool DMA = SA::DMA;
  __shared__ __attribute__((aligned(16))) char ta[SUM ? 16 : SA::BYTES];
  __shared__ __attribute__((aligned(16))) char buf0[SA::BYTES + SX::BYTES];      // B, X
  __shared__ __attribute__((aligned(16))) char buf1[DMA ? SA::BYTES + SX::BYTES : 16];
  __shared__ uint4 tp[SUM ? 1 : NF * NC * 64];
  __shared__ __attribute__((aligned(16))) float rx[C];      // cu a^(n - 1 - r + shift): of row r in the state's sum

  // Workgroup i runs on XCD i % 8, each with its own L2: the jobs and column tiles of a segment, which read the same rows, are
  // given to one of them.  (Heads that share a key head are segments of their own, on any of them.  8 x 2048 tokens, 16 heads of 64 on 16
  // key heads 47 us, on four 45.)
  uint32_t item = blockIdx.x / args.per, rest = blockIdx.x - item * args.per;
  if (args.by_xcd) {
    const uint32_t k = blockIdx.x >> 3, o = k / args.per;
    rest = k - o * args.per;
    item = o * 8 + (blockIdx.x & 7);
    if (item >= (uint32_t)args.items) return;
  }
  int ji = 0;
  while (rest >= (uint32_t)args.job[ji].xtiles) rest -= (uint32_t)args.job[ji++].xtiles;
  const LaJob& j = args.job[ji];
  const int xt = (int)rest, unit = (int)(item / (uint32_t)args.nseg), seg = (int)(item - (uint32_t)unit * (uint32_t)args.nseg);
  if (SUM && seg == args.nseg - 1) return;      // no segment has its sum in front of it
  const int b = unit / args.H, h = unit - b * args.H;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, g = lane >> 4;
  const int live = ca_len(args.lens, args.lens64, b, args.L);
  const bool back = j.back != 0;
  const int x0 = xt * XT, xc = x0 + 16 * wave;      // first column of the workgroup, of the wave

  const float gd = la_log_decay(args.log_decay, h);
  // factors of pairs of tiles by the lane's rows: on the diagonal (zero above it), one tile apart, 16 more rows; of what the
  // state gives a row
  float wd[4], w1[4], w16 = 0.f, wy[KT];
  if constexpr (!SUM) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int gap = li - 4 * g - r;
      wd[r] = gap >= 0 ? j.cp * expf(gd * (float)gap) : 0.f;
      w1[r] = j.cp * expf(gd * (float)(gap + 16));
    }
    w16 = expf(gd * 16.f);
#pragma unroll
    for (int u = 0; u < KT; ++u) wy[u] = j.ci * expf(gd * (float)(16 * u + li + 1 - j.shift));
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
  const int da = j.da, dx = j.dx;
  const int64_t state = (int64_t)da * dx;
  // byte offset of tile m's row r of the lane's column in a state, past its end where there is none
  auto place = [&](int m, int r, int sr, int sc) __attribute__((always_inline)) {
    const int d = 32 * (m >> 1) + 8 * g + 4 * (m & 1) + r, at = (d * sr + (xc + li) * sc) * 4;
    return d < da && xc + li < dx ? at : (int)SA::NONE;
  };
#pragma unroll
  for (int m = 0; m < NS; ++m) s[m] = caf4{0.f, 0.f, 0.f, 0.f};
  if constexpr (!SUM) {
    // few segments: the state in front of this one from the sums of those before it; many: as la_prefix_kernel left it
    auto add = [&](const float* p, int sr, int sc, float an, float less) __attribute__((always_inline)) {
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)state * 4, kRawBufferWord3);
      float v[NS][4];
#pragma unroll
      for (int m = 0; m < NS; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) v[m][r] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, place(m, r, sr, sc), 0, 0));
#pragma unroll
      for (int m = 0; m < NS; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[m][r] = la_decayed(s[m][r], an, less) + v[m][r];
    };
    const float* sums = j.seg + (int64_t)unit * args.nseg * state;
    const bool few = args.nseg <= LA_FEW_SEGMENTS;
    if (few && j.s0) add(j.s0 + unit * state, j.s_r, j.s_c, 0.f, 0.f);
    if (!few) add(sums + seg * state, j.dx, 1, 0.f, 0.f);
    else
      for (int k = 0; k < seg; ++k) {
        const int64_t t0 = (int64_t)(back ? args.nseg - 1 - k : k) * args.seg_tokens, m = live - t0;
        const float n = (float)(m < 0 ? 0 : m > args.seg_tokens ? args.seg_tokens : m);
        add(sums + k * state, j.dx, 1, expf(gd * n), expm1f(gd * n));
      }
  }

  const int64_t base_a = (b * j.a.sb + (h / j.a.group) * j.a.sh) * ESZ, base_b = (b * j.b.sb + (h / j.b.group) * j.b.sh) * ESZ,
                base_x = (b * j.x.sb + (h / j.x.group) * j.x.sh + x0) * ESZ;
  const char *pa = j.a.p + base_a, *pb = j.b.p + base_b, *px = j.x.p + base_x;
  const int sa_b = (int)j.a.sl * ESZ, sb_b = (int)j.b.sl * ESZ, sx_b = (int)j.x.sl * ESZ;      // bytes between tokens
  const int ysz = j.y32 ? 4 : ESZ, yrow = args.H * dx * ysz;
  const bool wanted = j.y != nullptr, wide = DT == HCLSM_F32 || j.y32 != 0, fine = NC == 3 || args.fine != 0;
  char* py = j.y + ((int64_t)b * args.L * args.H + h) * dx * ysz;
  const float cu = j.cu;
  const int shift = j.shift;
  SA ra, rb;
  SX rxs;
  auto tokens = [&](int k, int& t0, int& n) __attribute__((always_inline)) {
    t0 = first + (back ? nch - 1 - k : k) * C;
    const int e = live < t_end ? live : t_end;
    n = e - t0;
    n = n < 0 ? 0 : n > C ? C : n;
  };
  auto load_a = [&](int t0, int n) __attribute__((always_inline)) {
    if constexpr (!SUM) ra.load(pa + (int64_t)t0 * sa_b, sa_b, n, da, back, ta, wave);
  };
  auto load_bx = [&](int t0, int n, char* t) __attribute__((always_inline)) {
    rb.load(pb + (int64_t)t0 * sb_b, sb_b, n, da, back, t, wave);
    rxs.load(px + (int64_t)t0 * sx_b, sx_b, n, dx - x0, back, t + SA::BYTES, wave);
  };
  auto pair = [](int f, int& tt, int& sp) __attribute__((always_inline)) {
    tt = KT == 4 ? (f < 2 ? f : 2 + ((f - 2) >> 1)) : f;
    sp = KT == 4 && f >= 2 ? (f & 1) : 0;
  };
  if constexpr (!SUM) {     // the tiles above the diagonal, beside those on it: zeros throughout
    if (wave < KT / 2)
#pragma unroll
      for (int p = 0; p < NC; ++p) reinterpret_cast<uint2*>(tp)[((3 * wave * NC + p) * 64 + lane) * 2 + 1] = uint2{0, 0};
  }
  int tab = -1;             // live tokens that rx and decay are for
  float decay = 0.f;
  bool slow = false;

  if (nch > 0) {
    int t0, n;
    tokens(0, t0, n);
    if (n > 0) {
      load_bx(t0, n, buf0);
      load_a(t0, n);
    }
  }
  auto work = [&](int k, char* tb, char* next) __attribute__((always_inline)) {
    int t0, n, t1 = 0, n1 = 0;
    tokens(k, t0, n);
    if (k + 1 < nch) tokens(k + 1, t1, n1);
    char* tx = tb + SA::BYTES;
    if constexpr (DMA) {
      ca_wait_vmem();
      la_barrier();         // the chunk is in LDS, and every wave is done with the one before
      if (n1 > 0) load_bx(t1, n1, next);
    } else {
      la_barrier();
      if (n > 0) {
        if constexpr (!SUM) ra.store(ta);
        rb.store(tb);
        rxs.store(tx);
      }
      if (n1 > 0) {
        load_bx(t1, n1, next);
        load_a(t1, n1);
      }
    }
    if (n != tab) {
      tab = n;
      if ((int)threadIdx.x < C)
        rx[threadIdx.x] = (int)threadIdx.x < n ? cu * expf(gd * (float)(n - 1 - (int)threadIdx.x + shift)) : 0.f;
      const float an = expf(gd * (float)n);      // (la_decayed, one of its two forms for all)
      slow = __builtin_amdgcn_readfirstlane(an >= 0.5f ? 1 : 0) != 0;
      decay = slow ? expm1f(gd * (float)n) : an;
      if constexpr (SUM && DMA) __syncthreads();
    }
    if constexpr (!DMA) la_barrier();

    caf4 y[SUM ? 1 : KT];
    if constexpr (!SUM) {
#pragma unroll
      for (int u = 0; u < KT; ++u) y[u] = caf4{0.f, 0.f, 0.f, 0.f};
      if (n > 0) {
        // weights of pairs: tile (s, t) leaves a lane with s = 4g + r of its t = li.  The ten tiles at or below the diagonal (three
        // of 32 tokens) are shared out as evenly as they go: two for every wave and a third for waves 0 and 1 (one for
        // waves 0 to 2); the operands of CG products of all a wave's tiles are read before the first.
        {
          constexpr int CG = DA == 64 ? 2 : NP == 1 ? 4 : 1, SUBS = KT == 4 ? 3 : 1, AS = KT == 4 ? 2 : 1;
          caf4 w[SUBS];
          int tt[SUBS], st[SUBS];
          bool mine[SUBS];
          if constexpr (KT == 4) {
            tt[0] = tt[1] = wave < 2 ? wave + 1 : 3;
            st[0] = wave < 3 ? 0 : 2;
            st[1] = st[0] + 1;
            tt[2] = st[2] = 2 * wave;
            mine[0] = mine[1] = true;
            mine[2] = wave < 2;
          } else {
            tt[0] = wave > 0 ? 1 : 0;
            st[0] = wave > 1 ? 1 : 0;
            mine[0] = wave < 3;
          }
#pragma unroll
          for (int o = 0; o < SUBS; ++o) w[o] = caf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c0 = 0; c0 < DA / 32; c0 += CG) {
            LaFrag fa[AS][CG][NP], fb[SUBS][CG][NP];
#pragma unroll
            for (int o = 0; o < SUBS; ++o)
              if (mine[o])
#pragma unroll
                for (int c = 0; c < CG; ++c)
#pragma unroll
                  for (int p = 0; p < NP; ++p) {
                    if (o != 1) fa[o >> 1][c][p] = TA::frag(ta + p * SA::PLANE, 16 * tt[o], c0 + c, li, g);
                    fb[o][c][p] = TA::frag(tb + p * SA::PLANE, 16 * st[o], c0 + c, li, g);
                  }
            ca_fence();
#pragma unroll
            for (int c = 0; c < CG; ++c)
#pragma unroll
              for (int i = 0; i < NP; ++i)
#pragma unroll
                for (int p = 0; p < NP; ++p)
                  if (i + p <= MOST) {
#pragma unroll
                    for (int o = 0; o < (KT == 4 ? 2 : 0); ++o) w[o] = LaB::mma(fb[o][c][i], fa[0][c][p], w[o]);
                  }
            if (mine[SUBS - 1])
#pragma unroll
              for (int c = 0; c < CG; ++c)
#pragma unroll
                for (int i = 0; i < NP; ++i)
#pragma unroll
                  for (int p = 0; p < NP; ++p)
                    if (i + p <= MOST) w[SUBS - 1] = LaB::mma(fb[SUBS - 1][c][i], fa[AS - 1][c][p], w[SUBS - 1]);
          }
          auto weigh = [&](int o) __attribute__((always_inline)) {
            const int apart = tt[o] - st[o];      // tiles between the two
            const float more = apart > 2 ? w16 * w16 : apart > 1 ? w16 : 1.f;
#pragma unroll
            for (int r = 0; r < 4; ++r)      // (what lies above the diagonal may be infinite)
              w[o][r] = 16 * apart + li >= 4 * g + r ? w[o][r] * (apart > 0 ? w1[r] * more : wd[r]) : 0.f;
            return KT == 4 ? (tt[o] < 2 ? tt[o] : 2 * tt[o] - 2 + (st[o] >> 1)) : tt[o];
          };
          if constexpr (KT == 4) {
            const int f = weigh(0);
            weigh(1);
            LaFrag fp[NC];
            la_split<NC>(w, fp);
#pragma unroll
            for (int p = 0; p < NC; ++p) tp[(f * NC + p) * 64 + lane] = __builtin_bit_cast(uint4, fp[p]);
          }
          if (mine[SUBS - 1]) {
            const int f = weigh(SUBS - 1);
            uint2 fp[NC];
            la_split<NC>(w[SUBS - 1], fp);
#pragma unroll
            for (int p = 0; p < NC; ++p) {
              reinterpret_cast<uint2*>(tp)[((f * NC + p) * 64 + lane) * 2 + (st[SUBS - 1] & 1)] = fp[p];
              asm volatile("" ::: "memory");      // (two writes in one instruction would wait for the transfers in flight)
            }
          }
        }
        // what the state gives: y^T = S^T A^T, the next operands on their way
        {
          LaFrag fa[2][KT][NP], fs[2][NC];
          auto get = [&](int c, LaFrag (*f)[NP]) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < KT; ++u)
#pragma unroll
              for (int p = 0; p < NP; ++p) f[u][p] = TA::frag(ta + p * SA::PLANE, 16 * u, c, li, g);
          };
          get(0, fa[0]);
          la_split<NC>(&s[0], fs[0]);
#pragma unroll
          for (int c = 0; c < DA / 32; ++c) {
            if (c + 1 < DA / 32) get(c + 1, fa[(c + 1) & 1]);
            ca_fence();
            la_mma_all<NC, NP, MOST, KT>(fs[c & 1], fa[c & 1], y);
            if (c + 1 < DA / 32) la_split<NC>(&s[2 * c + 2], fs[(c + 1) & 1]);
            ca_fence();
          }
        }
#pragma unroll
        for (int u = 0; u < KT; ++u) y[u] *= wy[u];
      }
      la_barrier();         // the weights are in LDS, and every wave is done with A
      if constexpr (DMA) {
        if (n1 > 0) load_a(t1, n1);
      }
    }
    LaFrag fx[KT / 2][NP];
    if (n > 0) {
#pragma unroll
      for (int sp = 0; sp < KT / 2; ++sp)
#pragma unroll
        for (int p = 0; p < NP; ++p) fx[sp][p] = TX::frag_t(tx + p * SX::PLANE, 32 * sp, wave, li, g);
      if constexpr (!SUM) {
        constexpr int ORDER[6] = {0, 1, 2, 4, 3, 5};      // products in a row have results of their own
        LaFrag fp[NF][NC];
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
          for (int p = 0; p < NC; ++p) fp[f][p] = ca_frag<HCLSM_BF16>(tp[(f * NC + p) * 64 + lane]);
        ca_fence();
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
          for (int p = 0; p < NC; ++p)
            if (i + p <= MOST)
#pragma unroll
              for (int o = 0; o < NF; ++o) {
                const int f = NF == 6 ? ORDER[o] : o;
                int tt, sp;
                pair(f, tt, sp);
                y[tt] = LaB::mma(fx[sp][i], fp[f][p], y[tt]);
              }
      }
    }
    if constexpr (!SUM) {      // (here, not at the end: the state's sum hides the stores)
      if (wanted) {
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(py + (int64_t)t0 * yrow, 0, 0x7fffffff, kRawBufferWord3);
        const int cb = xc + 4 * g < dx ? (xc + 4 * g) * ysz : (int)SA::NONE;
        auto put_all = [&](auto put) __attribute__((always_inline)) {
          if (n == C) {
            const int off = cb < 0 ? cb : (back ? 15 - li : li) * yrow + cb;
#pragma unroll
            for (int u = 0; u < KT; ++u) put(y[u], rs, off, (back ? KT - 1 - u : u) * 16 * yrow);
          } else {      // tokens that are not live get zeros
#pragma unroll
            for (int u = 0; u < KT; ++u) {
              const int r = 16 * u + li, tok = r < n && back ? n - 1 - r : r;
              put(r < n ? y[u] : caf4{0.f, 0.f, 0.f, 0.f}, rs, cb >= 0 && t0 + tok < t_end ? tok * yrow + cb : (int)SA::NONE, 0);
            }
          }
        };
        if (wide)
          put_all([](caf4 v, __amdgpu_buffer_rsrc_t rs, int off, int so) __attribute__((always_inline)) {
            typedef uint32_t u4 __attribute__((ext_vector_type(4)));
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, v), rs, off, so, 0);
          });
        else if constexpr (DT != HCLSM_F32)
          put_all([](caf4 v, __amdgpu_buffer_rsrc_t rs, int off, int so) __attribute__((always_inline)) {
            typedef uint32_t u2 __attribute__((ext_vector_type(2)));
            __builtin_amdgcn_raw_buffer_store_b64(u2{CaT<DT>::pack2(v[0], v[1]), CaT<DT>::pack2(v[2], v[3])}, rs, off, so, 0);
          });
      }
    }
    if (n > 0) {
      // the state behind the chunk
      if (slow) {
#pragma unroll
        for (int m = 0; m < NS; ++m)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[m][r] = fmaf(s[m][r], decay, s[m][r]);
      } else {
#pragma unroll
        for (int m = 0; m < NS; ++m) s[m] *= decay;
      }
#pragma unroll
      for (int sp = 0; sp < KT / 2; ++sp) {
        float v[8];
        const caf4 w0 = *reinterpret_cast<const caf4*>(rx + 32 * sp + 4 * g), w1 = *reinterpret_cast<const caf4*>(rx + 32 * sp + 16 + 4 * g);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float x = 0.f;
#pragma unroll
          for (int p = NP - 1; p >= 0; --p) x += (float)fx[sp][p][e];
          v[e] = x * (e < 4 ? w0[e & 3] : w1[e & 3]);      // (rows that are not live are zeros)
        }
        if (fine) la_update<DA, NP, 3, SA::PLANE>(tb, 32 * sp, v, s, li, g);
        else la_update<DA, NP, 2, SA::PLANE>(tb, 32 * sp, v, s, li, g);
      }
    }
  };
  if constexpr (DMA) {
    for (int k = 0; k < nch; k += 2) {
      work(k, buf0, buf1);
      if (k + 1 < nch) work(k + 1, buf1, buf0);
    }
  } else {
    for (int k = 0; k < nch; ++k) work(k, buf0, buf0);
  }

  float* out = SUM ? j.seg + ((int64_t)unit * args.nseg + seg) * state
                   : seg == args.nseg - 1 && j.s1 ? j.s1 + unit * state : nullptr;
  if (out != nullptr) {
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(out, 0, (int)state * 4, kRawBufferWord3);
    const int sr = SUM ? j.dx : j.s_r, sc = SUM ? 1 : j.s_c;
#pragma unroll
    for (int m = 0; m < NS; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(s[m][r]), rs, place(m, r, sr, sc), 0, 0);
  }
}

template <int DT, int DA> int la_launch_one(const LaArgs& a, bool sum, hipStream_t st) {
  const dim3 grid((a.by_xcd ? (a.items + 7) / 8 * 8 : a.items) * a.per), block(LA_THREADS);
  if (sum) hipLaunchKernelGGL((la_kernel<DT, DA, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((la_kernel<DT, DA, false>), grid, block, 0, st, a);
  HCLSM_LAUNCH_CHECK();
  return 0;
}

template <int DT> int la_launch(const LaArgs& a, int da, bool sum, hipStream_t st) {
  if (da == 64) return la_launch_one<DT, 64>(a, sum, st);
  if (da == 128) return la_launch_one<DT, 128>(a, sum, st);
  return la_launch_one<DT, 256>(a, sum, st);
}

}  // namespace hclsm
