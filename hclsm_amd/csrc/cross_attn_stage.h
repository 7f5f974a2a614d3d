// Moving rows of heads into LDS and operand registers, for the cross-attention kernels.
#pragma once

#include "cross_attn.h"

namespace hclsm {

// Transfer of a tile of ROWS rows from global memory straight to LDS (16 bytes per lane to consecutive LDS addresses of
// a wave; which chunk of which row that is, is chosen by the lane's global address), one tile ahead of its use.  A
// chunk's offset from the tile's first row does not change from tile to tile; rows past the end, chunks past dh and the
// layout's padding get an offset past the buffer resource's end, for which the hardware writes zeros.
template <int DT, int DH, int NT, int ROWS> struct CaStage {
  using A = CaT<DT>;
  using Tile = CaTile<DT, DH>;
  static constexpr int BYTES = Tile::bytes(ROWS, NT), N = BYTES / (NT * 16);
  static constexpr int ESZ = (int)sizeof(typename A::T);
  static constexpr uint32_t NONE = 0xffffffffu;
  uint32_t off[N];

  static __device__ __forceinline__ int row(int n) { return ((int)threadIdx.x + n * NT) / Tile::PC; }
  static __device__ __forceinline__ int chunk(int n) { return (((int)threadIdx.x + n * NT) % Tile::PC) ^ Tile::swap(row(n)); }

  // rows one stride apart
  __device__ __forceinline__ void init(int64_t stride, int dh) {
#pragma unroll
    for (int n = 0; n < N; ++n)
      off[n] = row(n) < ROWS && chunk(n) * A::EPC < dh ? (uint32_t)row(n) * (uint32_t)(stride * ESZ) + chunk(n) * 16 : NONE;
  }
  // rows of a unit, the first one being head `phase` of its query: `used` rows of a tile
  __device__ __forceinline__ void init_rows(const CaArgs& a, int64_t sl, int64_t sh, int phase, int used) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      int qi, hg;
      ca_row(a, phase + row(n), qi, hg);
      off[n] = row(n) < used && chunk(n) * A::EPC < a.dh
                   ? (uint32_t)qi * (uint32_t)(sl * ESZ) + (uint32_t)hg * (uint32_t)(sh * ESZ) + chunk(n) * 16 : NONE;
    }
  }
  // base: first row of the tile; n_rows: rows there are from it on; wave: index of the wave, in a scalar register
  __device__ __forceinline__ void load(const char* base, int n_rows, char* t, int wave) const {
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 0x7fffffff, kRawBufferWord3);
    if (n_rows >= ROWS) {
#pragma unroll
      for (int n = 0; n < N; ++n)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (ca_lds_void*)(t + (n * NT + wave * 64) * 16), 16, (int)off[n], 0, 0, 0);
    } else {
#pragma unroll
      for (int n = 0; n < N; ++n)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (ca_lds_void*)(t + (n * NT + wave * 64) * 16), 16,
                                                 (int)(row(n) < n_rows ? off[n] : NONE), 0, 0, 0);
    }
  }
  // zeros for the rows whose bit is clear: what a masked row holds (NaN included) never reaches a product
  static __device__ __forceinline__ void drop(char* t, uint64_t live) {
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (row(n) < ROWS && !(live >> (row(n) & 63) & 1))
        *reinterpret_cast<uint4*>(t + ((int)threadIdx.x + n * NT) * 16) = uint4{0, 0, 0, 0};
  }
};

// This wave's transfers are in LDS (gfx9 encoding of s_waitcnt with the vector-memory count alone).
__device__ __forceinline__ void ca_wait_vmem() { __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8)); }
// No instruction moves across: operand reads stay ahead of the products they are to overlap with.
__device__ __forceinline__ void ca_fence() { __builtin_amdgcn_sched_barrier(0); }

// A row's operand fragments straight from global memory (zeros past dh and for rows that are not live).
template <int DT, int DH> __device__ __forceinline__ void ca_row_frags(const char* p, int g, int dh, bool live, uint4* f) {
  using A = CaT<DT>;
#pragma unroll
  for (int c = 0; c < DH / A::KS; ++c) {
    const int e = (4 * c + g) * A::EPC;
    f[c] = uint4{0, 0, 0, 0};
    if (live && e < dh) f[c] = *reinterpret_cast<const uint4*>(p + e * (int)sizeof(typename A::T));
  }
}

}  // namespace hclsm
