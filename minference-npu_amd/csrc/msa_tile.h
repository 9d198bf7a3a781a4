// Rows from global memory to MFMA operands, through LDS.
//
// An MFMA operand wants 16 rows in 16 neighbouring lanes, 16 bytes of each: read
// like that from global memory every lane of a pass touches another cache line,
// which the L1 serves slowly at most row strides (the weight sums' stats pass of 16
// heads x 16384 x 128 read in place: 1000 us; through LDS, shared by four waves:
// 580).  Here a wave loads whole rows, neighbouring lanes on
// neighbouring 16 bytes, into registers, later writes them to LDS, and reads
// operands back.  The 16-byte chunks of a row are permuted by its number so that
// neither side has bank conflicts: 16 lanes that read one chunk of 16 rows hit
// 16 different 16-byte bank groups.
#pragma once

#include "msa_common.h"

namespace msa {

template <int D, int ROWS>
struct Tile {
  static constexpr int NCH = D / 8;               // 16-byte chunks of a row
  static constexpr int NL = ROWS * NCH / 64;      // loads of a lane
  static constexpr int BYTES = ROWS * D * 2;
  static_assert(ROWS * NCH % 64 == 0, "a tile is whole wave loads");

  // Place of chunk c of row r.  8 chunks: two rows fill the banks, so pairs of
  // rows take turns; 12: rows start 12 bank groups apart, so four rows take every
  // fourth group and groups of four rows take turns among them, such that groups
  // 0 and 3 of one chunk and 1 and 2 of the next do not meet either (an operand read
  // takes its lanes in this order); 16 and more: every row its own permutation.
  __device__ static int place(int r, int c) {
    if constexpr (NCH == 8) return r * 8 + (c ^ ((r >> 1) & 7));
    else if constexpr (NCH == 12) {
      const int g = (r >> 2) & 3;
      return r * 12 + (c & ~3) + ((((c & 1) << 1) | ((c >> 1) & 1)) ^ g ^ (g >> 1));
    } else return r * NCH + (c ^ (r & 15));
  }

  uint32_t off[NL];    // byte offset of this lane's i-th chunk from the tile's first row
  uint32_t put[NL];    // its place in LDS, bytes

  __device__ Tile(int lane, uint32_t stride) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int f = 64 * i + lane, r = f / NCH, c = f - r * NCH;
      off[i] = uint32_t(r) * stride + 16u * c;
      put[i] = 16u * place(r, c);
    }
  }

  // AUX: cache policy.  soff: bytes from the descriptor's base to the tile,
  // inside the descriptor; rows behind its end read 0.
  template <int AUX>
  __device__ void load(__amdgpu_buffer_rsrc_t rs, uint32_t soff, u32x4 (&x)[NL]) const {
#pragma unroll
    for (int i = 0; i < NL; ++i)
      x[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, off[i], soff, AUX));
  }

  // The same without a scalar offset: base may lie behind the descriptor's end.
  __device__ void load_at(__amdgpu_buffer_rsrc_t rs, uint32_t base, u32x4 (&x)[NL]) const {
#pragma unroll
    for (int i = 0; i < NL; ++i)
      x[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, base + off[i], 0, 0));
  }

  __device__ void store(unsigned char* lds, const u32x4 (&x)[NL]) const {
#pragma unroll
    for (int i = 0; i < NL; ++i) *reinterpret_cast<u32x4*>(lds + put[i]) = x[i];
  }

  // Operand of rows 16 u + lc, dims 32 ks + 8 lr .. +7.
  __device__ static u32x4 operand(const unsigned char* lds, int u, int lc, int lr, int ks) {
    return *reinterpret_cast<const u32x4*>(lds + 16 * place(16 * u + lc, 4 * ks + lr));
  }
};

// What a wave wrote to LDS for itself is there for its later reads (LDS
// serves a wave in order); this keeps the compiler from moving them.
__device__ inline void wave_lds_fence() {
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
}

}  // namespace msa
