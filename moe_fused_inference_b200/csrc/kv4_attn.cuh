// kv4_attn.cuh — what the two attention kernels over the paged 4-bit KV cache
// share (kv4_attn.cu: few rows; kv4_prefill.cu: many).
#pragma once
#include "kv4.cuh"

namespace mfi {
namespace kv4 {

struct AttnArgs {
  const void* q;
  long long q_row, q_head;   // strides in elements
  const uint8_t* pool;
  const int* table;          // (n_seq, width)
  long long table_ld;
  const int* kv_lens;
  const int* cu_q;           // (n_seq + 1) or null: max_q rows each
  void* out;                 // (T, Hq, D)
  int* err;
  unsigned* counters;        // kCounterBytes
  float* part;               // few_bytes or many_bytes
  int T, max_q, n_seq, Hq, Hkv, page, num_pages, width;
  int few;                   // sequences of up to this many vectors (rows x heads of a group) are `few`
  bool many;                 // there may be others: the kernel for many rows follows
  bool q_vec;                // every query row starts on a 16-byte boundary
  int tpp_shift;             // log2 of the tiles of a page, -1 if that is no power of two
  float scale;
};

// Rows and tokens of sequence i, clamped to the query rows and the table.
struct Seq {
  int row0, rows, len;
};
__device__ __forceinline__ Seq sequence(const AttnArgs& a, int i) {
  Seq s;
  s.row0 = a.cu_q ? a.cu_q[i] : i * a.max_q;
  const int end = a.cu_q ? a.cu_q[i + 1] : s.row0 + a.max_q;
  s.rows = end - s.row0;
  s.len = a.kv_lens[i];
  const long long room = (long long)a.width * a.page;
  if (s.row0 < 0 || s.rows < 0 || end > a.T || s.rows > a.max_q) {
    report(a.err, kv4::kErrPage);
    s.rows = 0;
  }
  if (s.len > room || s.len < 0) {
    report(a.err, kv4::kErrPage);
    s.len = s.len < 0 ? 0 : int(room);
  }
  return s;
}


constexpr int kSms = 148;
constexpr int kCtas = kSms;                // of the kernel for many rows
constexpr int kFewCtas = 3 * kSms;         // most of the kernel for few rows
// Words of the workspace's head.  Few rows: two per CTA for the groups that begin
// with it, one for the pieces; every call takes them back to zero.  Many rows: the
// next item, one per part and warp; a CTA that gives up a wait leaves some of them
// behind, so the kernel for few rows, which runs first in every call, zeroes them.
constexpr int kItemCounter = 3 * kFewCtas, kPartCounters = kItemCounter + 1;
constexpr int kManyCounters = 1 + 8 * kCtas;
constexpr size_t kCounterBytes = 16384;
static_assert(kCounterBytes >= (kItemCounter + kManyCounters) * sizeof(unsigned), "room for the counters");
constexpr int kFew = 64;                   // vectors of a sequence and KV head that are few rows

// Bytes of the sums that parts of a piece or item leave for each other.
constexpr size_t few_bytes(int D) { return size_t(kFewCtas) * 2 * 16 * (D + 4) * sizeof(float); }
constexpr size_t many_bytes(int D) { return size_t(kCtas) * 256 * (D + 2) * sizeof(float); }

__device__ __forceinline__ uint32_t half_of(uint32_t w, int i) { return i ? w >> 16 : w & 0xFFFFu; }
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// E8M0 codes (nb bytes) to fp32; 255 gives NaN.
template <int nb>
__device__ __forceinline__ void codes(uint32_t w, float (&f)[nb]) {
#pragma unroll
  for (int i = 0; i < nb / 2; ++i) {
    uint32_t r;
    asm("cvt.rn.bf16x2.ue8m0x2 %0, %1;" : "=r"(r) : "h"(uint16_t(i ? w >> 16 : w)));
    f[2 * i] = __uint_as_float(r << 16);
    f[2 * i + 1] = __uint_as_float(r & 0xFFFF0000u);
  }
}
__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// 8 elements of a query row as they are; vec: p is 16-byte aligned.
template <class E>
__device__ __forceinline__ uint4 q8(const E* p, bool vec) {
  if (vec) return __ldg(reinterpret_cast<const uint4*>(p));
  const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
  return make_uint4(h[0] | uint32_t(h[1]) << 16, h[2] | uint32_t(h[3]) << 16,
                    h[4] | uint32_t(h[5]) << 16, h[6] | uint32_t(h[7]) << 16);
}
template <class E>
__device__ __forceinline__ float2 two_floats(uint32_t w);
template <>
__device__ __forceinline__ float2 two_floats<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <>
__device__ __forceinline__ float2 two_floats<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

// Whether a vector whose running maximum is m has left what the tensor cores' form
// holds, and is taken by attend_exactly instead: s qs - m in one rounding keeps what m
// has lost in its own, from 2^24 on more than a weight's exponent holds.  Infinity: a
// part of the vector asks for it (a NaN or an infinity in the scores does not).
__device__ __forceinline__ bool out_of_range(float m) { return fabsf(m) > 0x1p20f && m != -INFINITY; }

// One vector (row `row`, head h, over the first `see` tokens of sequence seq) by one
// warp on the CUDA cores, in fp32 throughout: for the few vectors whose operands or
// weights leave fp16 (out_of_range, values far stronger than those that the row sees).
// Some 60 instructions a token.
template <class E, int D>
__device__ __forceinline__ void attend_exactly(const AttnArgs& a, int seq, int row, int h, int see) {
  constexpr int nb = D / 32, kE = D / 32;  // channels of a lane
  const int lane = threadIdx.x & 31, el = kE * lane, b = el / 32, i = el % 32;
  const int key_at = ((i / 8) * nb + b) * 4 + (i % 8) / 2, value_at = ((i / 4) * nb + b) * 2 + (i % 4) / 2;
  const int tpp = a.page / kTile, g = h / (a.Hq / a.Hkv);
  const E* src = static_cast<const E*>(a.q) + (long long)row * a.q_row + h * a.q_head + el;
  float q[kE], o[kE], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int e = 0; e < kE; ++e) {
    q[e] = float(src[e]) * a.scale * 1.44269504088896341f;
    o[e] = 0.0f;
  }
  // elements of the lane at p, times s: a nibble's low bits are an exponent and one bit
  // of a significand, subnormal at 0
  auto elements = [](const uint8_t* p, float s, float (&x)[kE]) {
    const uint32_t w = kE == 4 ? *reinterpret_cast<const uint16_t*>(p) : *p;
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      const float y = __uint_as_float(((w >> (4 * e)) & 7u) << 22) * 0x1p126f;
      x[e] = ((w >> (4 * e)) & 8u ? -y : y) * s;
    }
  };
  constexpr int kRun = 4;  // tokens on their way at once, of one tile
#pragma unroll 1
  for (int t = 0; t < see; t += kRun) {
    const int tile = t / kTile;
    int id = __ldg(a.table + seq * a.table_ld + tile / tpp);
    if (unsigned(id) >= unsigned(a.num_pages)) id = 0;  // reported where its tiles are brought in
    const uint8_t* p = a.pool + ((uint64_t(unsigned(id)) * unsigned(a.Hkv) + unsigned(g)) * unsigned(tpp) +
                                 unsigned(tile % tpp)) * tile_bytes(D);
    float v[kRun][kE], x[kRun], top = m;
#pragma unroll
    for (int n = 0; n < kRun; ++n) {
      const int r = (t + n) % kTile;
      const uint8_t* c = p + 16 * D + r * nb + b;
      float k[kE];
      elements(p + r * (D / 2) + key_at, code_value(c[0]), k);
      elements(p + 8 * D + r * (D / 2) + value_at, code_value(c[D / 2]), v[n]);
      x[n] = 0.0f;
#pragma unroll
      for (int e = 0; e < kE; ++e) x[n] = fmaf(q[e], k[e], x[n]);
    }
#pragma unroll
    for (int n = 0; n < kRun; ++n) {
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) x[n] += __shfl_xor_sync(0xffffffffu, x[n], off);
      if (t + n < see) top = fmaxf(top, x[n]);
    }
    const float f = top == -INFINITY ? 1.0f : ex2(m - top);
    m = top;
    l *= f;
#pragma unroll
    for (int e = 0; e < kE; ++e) o[e] *= f;
#pragma unroll
    for (int n = 0; n < kRun; ++n) {
      if (t + n < see) {  // what a row does not see is not multiplied by zero: it may be NaN
        const float w = ex2(x[n] - (m == -INFINITY ? 0.0f : m));
        l += w;
#pragma unroll
        for (int e = 0; e < kE; ++e) o[e] = fmaf(w, v[n][e], o[e]);
      }
    }
  }
  __align__(8) E y[kE];
#pragma unroll
  for (int e = 0; e < kE; ++e) y[e] = E(l == 0.0f ? 0.0f : o[e] / l);
  E* dst = static_cast<E*>(a.out) + ((long long)row * a.Hq + h) * D + el;
  if (kE == 4) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(y);
  else *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(y);
}

}  // namespace kv4

// Launch the kernel for many rows on the sequences of more than a.few vectors.
cudaError_t launch_kv4_prefill(const kv4::AttnArgs& a, bool bf16, int D, cudaStream_t s);

}  // namespace mfi
