// Linear attention with a decay for each head: arguments shared by its kernels and their dispatch.
//
// State (da x dx, float32) and output of one head, a = exp(log_decay):
//     S_t = a S_{t-1} + k_t v_t^T,      o_t = c q_t^T S_t.
// A chunk of n tokens behind the state S of the tokens before it:
//     o_t = c sum_{s <= t} a^(t-s) (q_t . k_s) v_s + c a^(t+1) q_t^T S,     S' = a^n S + sum_s a^(n-1-s) k_s v_s^T.
// With D the gradient of S' (what reaches it from later tokens), go the gradient of o:
//     dq_t = c sum_{s <= t} a^(t-s) (go_t . v_s) k_s + c a^(t+1) S go_t
//     dv_s = c sum_{t >= s} a^(t-s) (k_s . q_t) go_t + a^(n-1-s) D^T k_s
//     dk_s = c sum_{t >= s} a^(t-s) (v_s . go_t) q_t + a^(n-1-s) D v_s,      D_before = a^n D + c sum_t a^(t+1) q_t go_t^T.
// All four are one job, the gradients of k and v on tokens taken backwards in time (row r of a chunk is token n-1-r):
//     y_r = cp sum_{s <= r} a^(r-s) (A_r . B_s) X_s + ci a^(r+1-shift) A_r S
//     S'  = a^n S + cu sum_s a^(n-1-s+shift) B_s X_s^T
//          A   B   X    state   cp ci cu  shift
//     o    q   k   v    S       c  c  1   0
//     dq   go  v   k    S^T     c  c  1   0
//     dv   k   q   go   D       c  1  c   1    backwards
//     dk   v   go  q    D^T     c  1  c   1    backwards
#pragma once

#include "cross_attn.h"

namespace hclsm {

constexpr int LA_MAX_DIM = 256;
// Up to LA_FEW_SEGMENTS the main kernel adds up the sums of the segments before its own (the last reads them all: at most seven
// states of up to 256 KB, from L2); beyond, a launch of la_prefix_kernel leaves each segment its state (10 us at 42 segments).
constexpr int LA_MAX_SEGMENTS = 256, LA_FEW_SEGMENTS = 8;

struct LaTensor {
  const char* p;
  int64_t sb, sl, sh;      // element strides
  int group;               // heads of the call that share one of this tensor's
};

struct LaJob {
  LaTensor a, b, x;
  char* y;                 // contiguous [B, L, H, dx]; null: not written
  const float* s0;         // [B, H] states, nullable (zeros)
  float* s1;               // states behind the last token, nullable
  float* seg;              // [B * H][nseg][da][dx]: sums of segments, then the states in front of them (nseg > 1)
  int s_r, s_c;            // element strides of a state's da and dx
  int da, dx, xtiles, shift, y32, back;
  float cp, ci, cu;
};

struct LaArgs {
  LaJob job[3];
  uint32_t per;            // workgroups of a segment: the column tiles of all jobs
  int items, by_xcd;       // B H nseg segments; whether they are dealt out to the XCDs
  int fine;                // the state is a result: its sums take X in three planes, not two
  const float* log_decay;  // [H]
  const void* lens;        // [B] live tokens, nullable
  int lens64, njobs;
  int B, H, L, nseg;
  int seg_tokens;          // tokens of a segment, whole chunks (nseg > 1)
};

// Tokens of a chunk: 64, or 32 where the planes (bf16: the two tiles) of wide heads would not fit the LDS.
constexpr int la_chunk(int dtype, int da) { return dtype == HCLSM_F32 || da > 128 || (dtype == HCLSM_F16 && da > 64) ? 32 : 64; }
// Sizes in between are multiplied as the next one.  8 x 2048 tokens, 16 heads, bf16, forward and with gradients: of 64 47 and 142 us; of 80
// 86 and 272, of 96 85 and 267, of 128 85 and 298; of 136 195 and 643, of 192 196 and 682, of 256 240 and 866.
constexpr int la_padded(int64_t d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }
constexpr int LA_THREADS = 256, LA_XT = 64;
// Waves per SIMD that the registers are to leave room for (the LDS holds no more workgroups).  bf16 heads of 128 with 3 spill their
// addresses, whose reloads wait for all transfers: 973 us for the 8 x 4096 tokens that take 746 with 2.
constexpr int la_waves(int dtype, int da) {
  return dtype == HCLSM_BF16 ? (da <= 64 ? 3 : 2) : da == 64 ? (dtype == HCLSM_F32 ? 3 : 2) : da == 128 ? 2 : 1;
}

// One launch of jobs that share a padded size (sum: the sums of segments alone).
int la_launch_f32(const LaArgs& a, int da, bool sum, hipStream_t st);
int la_launch_bf16(const LaArgs& a, int da, bool sum, hipStream_t st);
int la_launch_f16(const LaArgs& a, int da, bool sum, hipStream_t st);

// The decay of a head as the kernels use it: -inf (no memory) as a number whose multiples stay finite.
__device__ __forceinline__ float la_log_decay(const float* g, int h) {
  const float v = g[h];
  return v < -1e30f ? -1e30f : v;
}

// a^n s from a^n and a^n - 1.  Near one as s + (a^n - 1) s: a rounded a^n would be off alike in every chunk of a long memory.
__device__ __forceinline__ float la_decayed(float s, float an, float less) { return an >= 0.5f ? fmaf(s, less, s) : s * an; }

}  // namespace hclsm
