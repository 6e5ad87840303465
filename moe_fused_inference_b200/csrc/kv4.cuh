// kv4.cuh — the paged 4-bit KV cache: layout, codes and bounds shared by its
// kernels (kv4.cu: write and read; kv4_attn.cu: attention).
//
// A key or value vector of one KV head (D = 64 or 128) is cut into blocks of
// 32 elements, each held as MXFP4: E2M1 nibbles and one E8M0 code.  The pool is
//   uint8 (pages, Hkv, page / 16, 17 D)
// one tile of 17 D bytes per 16 consecutive tokens of a page and head:
//   [0, 8D)          16 key rows of D/2 bytes
//   [8D, 16D)        16 value rows of D/2 bytes
//   [16D, 16D + D/2) 16 rows of key codes, D/32 bytes each
//   [16D + D/2, 17D) 16 rows of value codes
// so that a tile, and any run of tiles of a page, is one contiguous piece of
// memory (17 D is a multiple of 64) that one bulk copy brings in.  Inside the
// rows the blocks are interleaved for the tensor cores' fragments: with nb =
// D / 32, the key row holds the 4-byte word t (elements 8t .. 8t+7) of block b
// as word t nb + b, the value row the 2-byte piece h (elements 4h .. 4h+3) of
// block b as piece h nb + b.  Nibbles are packed LSB-first.
//
// Block exponent e = ceil(log2(max(amax / 6, 1e-30))) as in mx_common.cuh, code
// e + 127 also for a block of zeros; a block with a value that is not finite
// holds code 255 and zeros, and reads as NaN.
#pragma once
#include "mx_common.cuh"

namespace mfi {
namespace kv4 {

constexpr int kTile = 16;  // tokens of a tile

__host__ __device__ constexpr int tile_bytes(int D) { return 17 * D; }

// Bytes of the pool's (page, head) piece.
__host__ __device__ constexpr long long head_bytes(int D, int page) {
  return (long long)(page / kTile) * tile_bytes(D);
}

// E8M0 code to its value, all 256 codes (0 is 2^-127, 255 is NaN).
__device__ __forceinline__ float code_value(uint32_t c) {
  return __uint_as_float(c == 255u ? 0x7FC00000u : (c == 0u ? 0x00400000u : c << 23));
}

// The four bytes of w, each two E2M1 values, to fp16x2 (low nibble: low half).
__device__ __forceinline__ void e2m1x8(uint32_t w, uint32_t (&o)[4]) {
  asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %4;\n"
      " cvt.rn.f16x2.e2m1x2 %0, a;\n cvt.rn.f16x2.e2m1x2 %1, b;\n"
      " cvt.rn.f16x2.e2m1x2 %2, c;\n cvt.rn.f16x2.e2m1x2 %3, d;\n}"
      : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3])
      : "r"(w));
}

// Device error codes of the cache's kernels.
constexpr int kErrPage = 11;  // page id, length or row range outside the pool, table or rows
constexpr int kErrSlot = 12;  // token slot past the pool

__device__ __forceinline__ void report(int* err, int code) { atomicCAS(err, 0, code); }

}  // namespace kv4
}  // namespace mfi
