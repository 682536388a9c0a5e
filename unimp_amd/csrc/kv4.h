// The 4-bit pages of a decode cache (include/unimp_hip.h, unimp_kv4_*): layout and element arithmetic shared by kv4.hip and kv4_attn.hip.
//
// A page = 32 tokens of one (layer, head), keys and values.  Elements are e2m1 codes; one E8M0 byte per (token, 32 consecutive dims): the MX block of
// the frozen towers' fp8 path (mx.hip) with 4-bit elements.  D dims, NB = ceil(D / 32) blocks (head dim 80: two whole blocks and one of 16 dims):
//   K codes   [0, 16 D)          block b at 512 b: token t's 16 bytes (8 in a 16-wide last block), dims in order, low nibble first.  A lane of
//                                v_mfma_scale_f32_16x16x128 (row r = l & 15, g = l >> 4) wants 32 consecutive k of its row, low nibble first: its
//                                fp4 operand is ONE 16-byte load of block g, token 16 tile + r.
//   V codes   [16 D, 32 D)       dword (g, c, i) = g D + c (D / 16) + i, g < 4, c < 16: nibble 4 h + e of it = token 16 h + 4 g + e, dim 16 i + c.
//                                The score tile's lane (query c, g) holds tokens 16 h + 4 g + e (h < 2, e < 4): p never changes lanes, and a lane's
//                                D / 16 operand dwords are consecutive bytes.
//   K scales  + 32 NB            byte 32 b + 2 (t & 15) + (t >> 4): the two tiles' scales of a lane are one 16-bit load
//   V scales  + 32 NB            byte 8 NB g + 8 b + 4 h + e
#pragma once
#include "common.h"

#define KV4_PAGE 32

__device__ __forceinline__ int kv4_nibble(int t) { return 4 * (t >> 4) + (t & 3); }      // token's nibble in its V dword

template <int D> struct Kv4 {
  static constexpr int NB = (D + 31) / 32, NI = D / 16, VOFF = 16 * D, KS = 32 * D, VS = 32 * D + 32 * NB, BYTES = 32 * D + 64 * NB;
  static constexpr int BLK_LAST = D - 32 * (NB - 1);                              // dims of the last block: 32 or 16
  static __device__ __forceinline__ int k_byte(int t, int b) { return 512 * b + t * (b == NB - 1 ? BLK_LAST / 2 : 16); }   // first byte of (token, block)
  static __device__ __forceinline__ int v_dword(int t, int d) { return VOFF + 4 * (((t >> 2) & 3) * D + (d & 15) * NI + (d >> 4)); }
  static __device__ __forceinline__ int ks_byte(int t, int b) { return KS + 32 * b + 2 * (t & 15) + (t >> 4); }
  static __device__ __forceinline__ int vs_byte(int t, int b) { return VS + 8 * NB * ((t >> 2) & 3) + 8 * b + kv4_nibble(t); }
};

// 2^(byte - 127); byte 255 (a block that held an infinity or a NaN): NaN.  Bytes written here are 2 ... 252 or 255.
__device__ __forceinline__ float kv4_scale(uint32_t byte) { return byte == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23); }
// block exponent from the exponent field of the block's largest magnitude (floor(log2 amax) + 127; 255: not finite): E8M0 byte, at least 2 so that no held
// value is subnormal
__device__ __forceinline__ int kv4_scale_byte(int eb) { return eb == 255 ? 255 : max(eb - 2, 2); }
