// kv4_attn.cu — attention over the paged 4-bit KV cache (layout: kv4.cuh).
//
// Sequence i owns the query rows cu_q[i] .. cu_q[i+1] - 1 (i max_q .. without
// cu_q) and the first kv_lens[i] tokens of the pages table[i]; its rows are
// the last of these tokens: row r of R sees tokens 0 .. L - R + r.
//   o = sum_p e^(s_p - m) v_p / sum_p e^(s_p - m),  s_p = scale q . k_p,  m = max s_p
// and zeros for a row that sees no token.
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "../../include/moe_fp4.h"
#include "kv4_attn.cuh"
#include "tc_ptx.cuh"
#include "tmap.cuh"
#include "work.cuh"

namespace mfi {

int kv4_check_pool(const void* pool, int Hkv, int D, int page, int num_pages);

namespace {

using namespace kv4;

// ---- few rows: up to 64 vectors a sequence and KV head, on mma.sync -------------
// A vector is one row of one query head; the R G vectors of a sequence and KV
// head (v = r G + h) are taken 8 kNT at a time (a "set").  The work is the list
// of all (sequence, KV head, set, tile of 16 tokens), in that order, short pieces
// padded; CTA c takes the c-th of `ctas` equal shares, whatever the lengths, and splits
// each piece (sequence, head, set) of its share over its warps.  8 or 16 vectors
// fill the n = 8 of mma.m16n8k16; an MMA of 64 or more would multiply zeros.
//
// What bounds it: the tile loop runs at 5.7 TB/s of the cache's bytes (232 warp
// instructions a tile of 4.25 bits an element, the conversions' pipe first), a call
// has some 14 us beside it: the launch, three dependent trips (lengths, page table,
// tiles), the join of the warps and of the CTAs.  4 KV heads of 128, 32 query
// heads, the cache not in L2: 1 sequence of 131072 tokens 27.6 us, 64 of up to 4096
// 31.6 us, 1 of 1152 11.8 us, 5 rows over 8191 tokens 14.6 us.  (The figures of the
// constants below are of one call over and over, its cache in L2, without the check of
// the maximum at the end, which costs up to 2%.)
//
// Per tile and warp, with mma.m16n8k16 (fp16 operands, fp32 sums):
//   S^T (16 tokens x 8 vectors) = K_b . Q_b^T for each block b of 32 elements,
//   the blocks joined by their codes: s = sum_b 2^(c_b - 127) S_b
//   O^T (D x 8 vectors) += V_b^T . P_b,  P_b = p 2^(c_b - 127)
// The E2M1 values are exact in fp16 and never multiplied by a scale: the codes
// go to the few scores and weights.  A stage's codes are turned into factors by
// one lane each and read back from shared memory.
// * The query rows are scaled by a power of two to a maximum in [2^14, 2^15),
//   which keeps all bits of a bf16 or fp16 row down to 2^-39 of its maximum; the key
//   factors by 2^-13, so that a score of keys up to 2^117 fits fp32.
// * p is rounded to fp16 (2^-12) after a factor 2^10, and multiplied by 2^(c_b -
//   top_b + 4), top_b the largest code that the warp has seen in block b of the
//   values: exact but for products below 2^-28 of the largest weight times the
//   block's largest scale, which lose bits and vanish below 2^-39; codes 29 and
//   more below top_b count as zero.  (One top for all blocks dropped channels
//   2^29 weaker than others.)
constexpr float kKeyUnit = 0x1p-13f;
// Tiles; 16, 32, 64: 64 sequences of up to 4096 tokens 31.6, 29.0, 32.8 us, three rows
// over 8191 tokens 12.8, 12.8, 15.3, 32 sequences of up to 2003 16.0, 17.2, 21.9.
constexpr unsigned kSnap = 32;
constexpr unsigned kLeast = 32;  // units of a piece at least
constexpr int kOneLevel = 16;    // parts; 8: three rows over 8191 tokens 14.7 instead of 12.8 us, 64: alike

template <int D, int kNT, int kPerSm>
struct Few {
  static constexpr int kWarps = kNT == 1 ? 12 / kPerSm : 8 / kPerSm;
  static constexpr int kChunk = 4;   // tiles of a pipeline stage
  // one read, one on its way; stages of 2 tiles 3 or 4 deep cost 2.6 and 3.3 us more
  // for 131072 tokens
  static constexpr int kStages = 2;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kVec = 8 * kNT;
  static constexpr int kStageBytes = kChunk * kv4::tile_bytes(D);
  static constexpr int kAcc = D + 4;                          // floats of a vector's sum: D, max, sum, pad
  static_assert(kVec * kAcc * 4 <= kStageBytes, "a warp's sums take the place of a stage");
  static constexpr int kFactors = kChunk * kv4::kTile * (D / 32) * 6;  // key factors fp32, value factors fp16
  static constexpr int kWarpBytes = kStages * kStageBytes + kFactors;
  static constexpr int kSmem = kWarps * kWarpBytes;
};

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same with sums that start at zero
__device__ __forceinline__ void mma16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                               uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
// Tiles of sequence s's pieces and their count of sets.
__device__ __forceinline__ int seq_tiles(const Seq& s) {
  return s.rows > 0 ? max(1, (s.len + kv4::kTile - 1) / kv4::kTile) : 0;
}

// Units of work of sequence s's pieces: their tiles, but kLeast at least, for a
// piece costs its start and joins (some 4 us) whatever its length.  With 1, 16, 32, 64
// units: 20 pieces of 1 tile 44.3, 7.4, 7.5, 7.5 us (with 1 they go to two CTAs one
// after the other), 16 sequences of 3000 tokens beside 8 empty ones 84.4, 19.1, 18.0,
// 18.7, 64 of up to 4096 34.3, 29.7, 29.0, 28.6.  Pieces of up to 2 kSnap units are
// never split, so only whole ones have units without tiles.
__device__ __forceinline__ int seq_units(const Seq& s) {
  return s.rows > 0 ? max(int(kLeast), seq_tiles(s)) : 0;
}
static_assert(kLeast <= 2 * kSnap, "padded pieces are not split");

// A warp's state: the running maximum (log2 domain) of each vector, the sum of
// its weights times 2^10, and block b of O^T times 2^(127 + 15 - top_b), top_b the
// block's largest value code plus one so far (a code of 255, NaN, counts as 0; two
// such neighbours may carry one too many): halves of top[b % 2].
template <int D, int kNT>
struct Running {
  uint32_t top[2];
  float m[kNT][2], l[kNT][2];
  float o[kNT][D / 16][4];
};

// What a warp knows of the thread's vectors: tokens that they see (lim), the
// power of two and scale that their scores lack (qs > 0), the query fragments.
// Tokens below `all` are seen by all vectors.
template <int D, int kNT>
struct Query {
  int all;
  int lim[kNT][2];
  float qs[kNT][2];
  uint32_t f[kNT][D / 16][2];
};

// kN tiles at `base` (shared memory), the first holding token `pos0`, of which
// tokens from `end` on count for nothing (their bytes may be anything);
// `factors`: this warp's place for their factors.
template <int D, int kNT, int kPerSm, int kN>
__device__ __forceinline__ void attend_tiles(Running<D, kNT>& w, const Query<D, kNT>& q,
                                             const uint8_t* base, uint8_t* factors, int pos0,
                                             int end) {
  constexpr int nb = D / 32;
  const int lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  // row r of the score tile is token (r & 1) * 4 + r / 2 (+ 8): the weights'
  // fragment then pairs tokens t and t + 4, so that the four lanes of a quad
  // read neighbouring value rows
  const int tok = (gid & 1) * 4 + (gid >> 1);
  float* kf = reinterpret_cast<float*>(factors);                          // [tile][token][block]
  uint32_t* vf = reinterpret_cast<uint32_t*>(factors + Few<D, kNT, kPerSm>::kChunk * kv4::kTile * nb * 4);  // [tile][pair][block]

  // ---- codes to factors.  Keys: one word a lane and turn.  Values: lane (tile,
  // pair) takes tokens t and t + 4, t = 0-3, 8-11
  __syncwarp();  // the previous tiles' factors are read
  {
    constexpr int kWords = kv4::kTile * nb / 4;  // words of a tile's key codes
#pragma unroll
    for (int k = 0; k < (kN * kWords + 31) / 32; ++k) {
      const int i = k * (32 / kWords) + lane / kWords, x = lane % kWords;
      if (kN * kWords % 32 == 0 || i < kN) {
        float f[4];
        codes<4>(*reinterpret_cast<const uint32_t*>(base + i * kv4::tile_bytes(D) + 16 * D + 4 * x), f);
        *reinterpret_cast<float4*>(kf + (i * kWords + x) * 4) =
            make_float4(f[0] * kKeyUnit, f[1] * kKeyUnit, f[2] * kKeyUnit, f[3] * kKeyUnit);
      }
    }
  }
  uint32_t ca = 0, cb = 0, t0 = w.top[0], t1 = w.top[1];
  const int ti = lane >> 3, pr = lane & 7, ta = pr < 4 ? pr : pr + 4;
  if (ti < kN) {
    const uint8_t* c = base + ti * kv4::tile_bytes(D) + 16 * D + D / 2 + ta * nb;
    if (nb == 4) {
      ca = *reinterpret_cast<const uint32_t*>(c);
      cb = *reinterpret_cast<const uint32_t*>(c + 16);
    } else {
      ca = *reinterpret_cast<const uint16_t*>(c);
      cb = *reinterpret_cast<const uint16_t*>(c + 8);
    }
    if (pos0 + ti * kv4::kTile + ta >= end) ca = 0;
    if (pos0 + ti * kv4::kTile + ta + 4 >= end) cb = 0;
    t0 = __vmaxu2(__vmaxu2(t0, (ca + 0x00010001u) & 0x00FF00FFu), (cb + 0x00010001u) & 0x00FF00FFu);
    t1 = __vmaxu2(__vmaxu2(t1, ((ca >> 8) + 0x00010001u) & 0x00FF00FFu), ((cb >> 8) + 0x00010001u) & 0x00FF00FFu);
  }
  // A NaN value block (rare) makes NaN of the vectors that see its token, whatever
  // the weight, and of no others: written here, left out of the products.
  const uint32_t bada = __vcmpeq4(ca, 0xFFFFFFFFu), badb = __vcmpeq4(cb, 0xFFFFFFFFu);
  if (uint32_t left = __ballot_sync(0xffffffffu, (bada | badb) != 0u)) {
    ca &= ~bada;
    cb &= ~badb;
    for (; left; left &= left - 1) {
      const int src = __ffs(left) - 1;
      const uint32_t a = __shfl_sync(0xffffffffu, bada, src), b = __shfl_sync(0xffffffffu, badb, src);
      const int pa = pos0 + __shfl_sync(0xffffffffu, ti * kv4::kTile + ta, src);
#pragma unroll
      for (int j = 0; j < kNT; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t bad = (pa < q.lim[j][i] ? a : 0u) | (pa + 4 < q.lim[j][i] ? b : 0u);
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            if ((bad >> (8 * (k / 2))) & 1u) w.o[j][k][i] = w.o[j][k][i + 2] = __uint_as_float(0x7FC00000u);
        }
    }
  }
  if (__any_sync(0xffffffffu, t0 != w.top[0] || t1 != w.top[1])) {
    t0 = __reduce_max_sync(0xffffffffu, t0 & 0xFFFFu) | __reduce_max_sync(0xffffffffu, t0 >> 16) << 16;
    t1 = __reduce_max_sync(0xffffffffu, t1 & 0xFFFFu) | __reduce_max_sync(0xffffffffu, t1 >> 16) << 16;
#pragma unroll
    for (int b = 0; b < nb; ++b) {
      const uint32_t now = half_of(b % 2 ? t1 : t0, b / 2), then = half_of(w.top[b % 2], b / 2);
      const float c = __uint_as_float(max(127 + int(then) - int(now), 0) << 23);
#pragma unroll
      for (int j = 0; j < kNT; ++j)
#pragma unroll
        for (int k = 2 * b; k < 2 * b + 2; ++k) {
          w.o[j][k][0] *= c;
          w.o[j][k][1] *= c;
          w.o[j][k][2] *= c;
          w.o[j][k][3] *= c;
        }
    }
    // Tokens that some vectors do not see yet, 2^24 stronger than others of their block
    // (rare): these vectors would lose what they see.  They are asked for once more.
    if (end > q.all) {
      bool far = false;
#pragma unroll
      for (int b = 0; b < nb; ++b) {
        const uint32_t then = half_of(w.top[b % 2], b / 2), now = half_of(b % 2 ? t1 : t0, b / 2);
        const uint32_t x = (ca >> (8 * b)) & 0xFFu, y = (cb >> (8 * b)) & 0xFFu;
        const uint32_t lo = min(then > 29u ? then - 1 : 255u, min(x > 28u ? x : 255u, y > 28u ? y : 255u));
        far |= now > max(then, lo + 24u);
      }
      if (__any_sync(0xffffffffu, far)) {
#pragma unroll
        for (int j = 0; j < kNT; ++j) w.m[j][0] = w.m[j][1] = INFINITY;
      }
    }
    w.top[0] = t0;
    w.top[1] = t1;
  }
  if (ti < kN) {
    float fa[nb], fb[nb];
    codes<nb>(ca, fa);
    codes<nb>(cb, fb);
    uint32_t h[nb];
#pragma unroll
    for (int b = 0; b < nb; ++b) {
      const float u = __uint_as_float((127 + 127 + 5 - half_of(w.top[b % 2], b / 2)) << 23);  // 2^(127 + 5 - top_b)
      h[b] = pack_half(fa[b] * u, fb[b] * u);
    }
    uint32_t* dst = vf + (ti * 8 + pr) * nb;
    if (nb == 4)
      *reinterpret_cast<uint4*>(dst) = make_uint4(h[0], h[1], h[nb - 2], h[nb - 1]);
    else
      *reinterpret_cast<uint2*>(dst) = make_uint2(h[0], h[1]);
  }
  __syncwarp();

  // ---- scores, without qs (which has the keys' 2^13)
  float s[kN][kNT][4];
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const uint8_t* tile = base + i * kv4::tile_bytes(D);
    uint32_t ka[nb], kb[nb];
    float fa[nb], fb[nb];
    if (D == 128) {
      const uint4 a = *reinterpret_cast<const uint4*>(tile + tok * 64 + tig * 16);
      const uint4 b = *reinterpret_cast<const uint4*>(tile + (tok + 8) * 64 + tig * 16);
      ka[0] = a.x; ka[1] = a.y; ka[nb - 2] = a.z; ka[nb - 1] = a.w;
      kb[0] = b.x; kb[1] = b.y; kb[nb - 2] = b.z; kb[nb - 1] = b.w;
      const float4 x = *reinterpret_cast<const float4*>(kf + (i * kv4::kTile + tok) * nb);
      const float4 y = *reinterpret_cast<const float4*>(kf + (i * kv4::kTile + tok + 8) * nb);
      fa[0] = x.x; fa[1] = x.y; fa[nb - 2] = x.z; fa[nb - 1] = x.w;
      fb[0] = y.x; fb[1] = y.y; fb[nb - 2] = y.z; fb[nb - 1] = y.w;
    } else {
      const uint2 a = *reinterpret_cast<const uint2*>(tile + tok * 32 + tig * 8);
      const uint2 b = *reinterpret_cast<const uint2*>(tile + (tok + 8) * 32 + tig * 8);
      ka[0] = a.x; ka[1] = a.y;
      kb[0] = b.x; kb[1] = b.y;
      const float2 x = *reinterpret_cast<const float2*>(kf + (i * kv4::kTile + tok) * nb);
      const float2 y = *reinterpret_cast<const float2*>(kf + (i * kv4::kTile + tok + 8) * nb);
      fa[0] = x.x; fa[1] = x.y;
      fb[0] = y.x; fb[1] = y.y;
    }
#pragma unroll
    for (int b = 0; b < nb; ++b) {
      uint32_t xa[4], xb[4];
      e2m1x8(ka[b], xa);
      e2m1x8(kb[b], xb);
#pragma unroll
      for (int j = 0; j < kNT; ++j) {
        float d[4];
        mma16816_first(d, xa[0], xb[0], xa[1], xb[1], q.f[j][2 * b][0], q.f[j][2 * b][1]);
        mma16816(d, xa[2], xb[2], xa[3], xb[3], q.f[j][2 * b + 1][0], q.f[j][2 * b + 1][1]);
        s[i][j][0] = b ? fmaf(d[0], fa[b], s[i][j][0]) : d[0] * fa[b];
        s[i][j][1] = b ? fmaf(d[1], fa[b], s[i][j][1]) : d[1] * fa[b];
        s[i][j][2] = b ? fmaf(d[2], fb[b], s[i][j][2]) : d[2] * fb[b];
        s[i][j][3] = b ? fmaf(d[3], fb[b], s[i][j][3]) : d[3] * fb[b];
      }
    }
  }
  const bool edge = pos0 + kN * kv4::kTile > min(q.all, end);  // tokens that not all vectors see
  if (edge) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int pa = pos0 + i * kv4::kTile + tok, pb = pa + 8;
#pragma unroll
      for (int j = 0; j < kNT; ++j) {
        const int l0 = min(q.lim[j][0], end), l1 = min(q.lim[j][1], end);
        if (pa >= l0) s[i][j][0] = -INFINITY;
        if (pa >= l1) s[i][j][1] = -INFINITY;
        if (pb >= l0) s[i][j][2] = -INFINITY;
        if (pb >= l1) s[i][j][3] = -INFINITY;
      }
    }
  }

  // ---- running maximum over the tiles' tokens
  float r0[kNT], r1[kNT];
#pragma unroll
  for (int j = 0; j < kNT; ++j) {
    float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      t0 = fmaxf(t0, fmaxf(s[i][j][0], s[i][j][2]));
      t1 = fmaxf(t1, fmaxf(s[i][j][1], s[i][j][3]));
    }
#pragma unroll
    for (int off = 4; off <= 16; off <<= 1) {
      t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, off));
      t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, off));
    }
    t0 *= q.qs[j][0];
    t1 *= q.qs[j][1];
    // the reference moves only when it is passed by more than 1 (p <= 2)
    const bool up0 = t0 > w.m[j][0] + 1.0f, up1 = t1 > w.m[j][1] + 1.0f;
    if (__any_sync(0xffffffffu, up0 || up1)) {
      // (sums of scores out of range are none: asked for once more)
      const float m0 = up0 ? (out_of_range(w.m[j][0]) ? INFINITY : t0) : w.m[j][0];
      const float m1 = up1 ? (out_of_range(w.m[j][1]) ? INFINITY : t1) : w.m[j][1];
      const float c0 = up0 ? ex2(w.m[j][0] - m0) : 1.0f, c1 = up1 ? ex2(w.m[j][1] - m1) : 1.0f;
      w.m[j][0] = m0;
      w.m[j][1] = m1;
      w.l[j][0] *= c0;
      w.l[j][1] *= c1;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        w.o[j][k][0] *= c0;
        w.o[j][k][1] *= c1;
        w.o[j][k][2] *= c0;
        w.o[j][k][3] *= c1;
      }
    }
    // a vector that has seen nothing keeps m = -inf; its scores are all -inf too
    r0[j] = (w.m[j][0] == -INFINITY ? 0.0f : w.m[j][0]) - 10.0f;
    r1[j] = (w.m[j][1] == -INFINITY ? 0.0f : w.m[j][1]) - 10.0f;
  }

  // ---- weights and values
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const uint8_t* tile = base + i * kv4::tile_bytes(D);
    uint32_t pf[kNT][nb][2];  // weights' fragments: tokens tig, tig + 4 (+ 8) of vector gid
    {
      uint32_t ga[nb], gb[nb];
      const uint32_t* src = vf + (i * 8 + tig) * nb;
      if (nb == 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(src), y = *reinterpret_cast<const uint4*>(src + 4 * nb);
        ga[0] = x.x; ga[1] = x.y; ga[nb - 2] = x.z; ga[nb - 1] = x.w;
        gb[0] = y.x; gb[1] = y.y; gb[nb - 2] = y.z; gb[nb - 1] = y.w;
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(src), y = *reinterpret_cast<const uint2*>(src + 4 * nb);
        ga[0] = x.x; ga[1] = x.y;
        gb[0] = y.x; gb[1] = y.y;
      }
#pragma unroll
      for (int j = 0; j < kNT; ++j) {
        const float p0 = ex2(fmaf(s[i][j][0], q.qs[j][0], -r0[j]));
        const float p1 = ex2(fmaf(s[i][j][1], q.qs[j][1], -r1[j]));
        const float p2 = ex2(fmaf(s[i][j][2], q.qs[j][0], -r0[j]));
        const float p3 = ex2(fmaf(s[i][j][3], q.qs[j][1], -r1[j]));
        w.l[j][0] += p0 + p2;
        w.l[j][1] += p1 + p3;
        const uint32_t pa = transpose8x8(pack_half(p0, p1)), pb = transpose8x8(pack_half(p2, p3));
#pragma unroll
        for (int b = 0; b < nb; ++b) {
          pf[j][b][0] = mul_half2(pa, ga[b]);
          pf[j][b][1] = mul_half2(pb, gb[b]);
        }
      }
    }
    // value rows tig, tig + 4, tig + 8, tig + 12: elements 4 gid .. 4 gid + 3 of each block
    uint32_t v[4][nb / 2];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint8_t* vr = tile + 8 * D + (tig + 4 * r) * (D / 2) + gid * (2 * nb);
      if (D == 128) {
        const uint2 x = *reinterpret_cast<const uint2*>(vr);
        v[r][0] = x.x;
        v[r][nb / 2 - 1] = x.y;
      } else {
        v[r][0] = *reinterpret_cast<const uint32_t*>(vr);
      }
    }
#pragma unroll
    for (int h = 0; h < nb / 2; ++h) {  // blocks 2h and 2h + 1
      constexpr uint32_t kLo = 0x0F0F0F0Fu;
      uint32_t a0[4], a1[4], a2[4], a3[4];
      e2m1x8((v[0][h] & kLo) | ((v[1][h] << 4) & ~kLo), a0);  // even elements, tokens t, t + 4
      e2m1x8(((v[0][h] >> 4) & kLo) | (v[1][h] & ~kLo), a1);  // odd elements
      e2m1x8((v[2][h] & kLo) | ((v[3][h] << 4) & ~kLo), a2);  // tokens t + 8, t + 12
      e2m1x8(((v[2][h] >> 4) & kLo) | (v[3][h] & ~kLo), a3);
#pragma unroll
      for (int j = 0; j < kNT; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k)  // byte k: block 2h + k / 2, elements 2 (k % 2), + 1
          mma16816(w.o[j][4 * h + k], a0[k], a1[k], a2[k], a3[k], pf[j][2 * h + (k >> 1)][0],
                   pf[j][2 * h + (k >> 1)][1]);
    }
  }
}

// Partial sums of a piece that several CTAs share: slot 0 of a CTA holds the
// piece that began before its share, slot 1 the one that goes on after it.
template <int D, int kNT, int kPerSm>
__device__ __forceinline__ float* slot_of(float* part, int cta, int slot) {
  return part + (size_t(cta) * 2 + slot) * (Few<D, kNT, kPerSm>::kVec * Few<D, kNT, kPerSm>::kAcc);
}

template <class E>
__device__ __forceinline__ void store_vector(const AttnArgs& a, const Seq& s, int g, int G, int v,
                                             int d0, const float (&o)[4], float inv, int D) {
  const int r = v / G, h = v - r * G;
  E* dst = static_cast<E*>(a.out) + ((long long)(s.row0 + r) * a.Hq + g * G + h) * D + d0;
  E x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = E(o[i] * inv);
  *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(x);
}

// Join what `count` warps or CTAs left of a set, each a row of kVec sums, read by
// `at`(i): this warp takes rows first, first + step, .. of all vectors at once.
template <int D, int kNT, int kPerSm, class At>
__device__ __forceinline__ void join_rows(int first, int step, int count, At at,
                                          float (&m)[Few<D, kNT, kPerSm>::kVec * D / 128],
                                          float (&l)[Few<D, kNT, kPerSm>::kVec * D / 128],
                                          float4 (&o)[Few<D, kNT, kPerSm>::kVec * D / 128]) {
  using F = Few<D, kNT, kPerSm>;
  constexpr int kPer = D / 4, kRows = 32 / kPer, kN = F::kVec / kRows;  // lanes of a vector, ..
  const int lane = threadIdx.x & 31, sub = lane / kPer, d0 = (lane % kPer) * 4;
#pragma unroll
  for (int k = 0; k < kN; ++k) {
    m[k] = -INFINITY;
    l[k] = 0.0f;
    o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
#pragma unroll 1
  for (int i = first; i < count; i += step) {
    const float* src = at(i) + sub * F::kAcc;
    float2 ml[kN];
    float4 x[kN];
#pragma unroll
    for (int k = 0; k < kN; ++k) {
      ml[k] = __ldcg(reinterpret_cast<const float2*>(src + k * kRows * F::kAcc + D));
      x[k] = __ldcg(reinterpret_cast<const float4*>(src + k * kRows * F::kAcc + d0));
    }
#pragma unroll
    for (int k = 0; k < kN; ++k) {
      const float nm = fmaxf(m[k], ml[k].x);
      const float ref = nm == -INFINITY ? 0.0f : nm;
      const float c0 = ex2(m[k] - ref), c1 = ex2(ml[k].x - ref);
      m[k] = nm;
      l[k] = l[k] * c0 + ml[k].y * c1;
      o[k].x = o[k].x * c0 + x[k].x * c1;
      o[k].y = o[k].y * c0 + x[k].y * c1;
      o[k].z = o[k].z * c0 + x[k].z * c1;
      o[k].w = o[k].w * c0 + x[k].w * c1;
    }
  }
}

// A CTA's part of a piece: tiles [t_lo, t_hi) of the set from vector v0 of KV
// head g of sequence seq.
struct Part {
  Seq s;
  int seq, g, v0, t_lo, t_hi, tiles;
  unsigned start, next;  // the piece's first unit, the first one after this part
};
struct Share {
  unsigned hi;           // the share's end
  unsigned units, ctas;  // CTA c takes units [c units / ctas, (c + 1) units / ctas)
};
// (x y - less) / d of 64 bits; in 32 where `units` of the call, times the CTAs, fit
__device__ __forceinline__ unsigned scaled(unsigned x, unsigned y, unsigned d, unsigned units,
                                           unsigned less = 0) {
  static_assert(kFewCtas < 512, "2^23 units times the CTAs fit 32 bits");
  return units < (1u << 23) ? (x * y - less) / d
                            : unsigned(((unsigned long long)x * y - less) / d);
}

template <class E, int D, int kNT, int kPerSm>
__global__ void __launch_bounds__(Few<D, kNT, kPerSm>::kThreads, kPerSm) kv4_attn_few_kernel(AttnArgs a) {
  using F = Few<D, kNT, kPerSm>;
  constexpr int nb = D / 32;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t s_bar[F::kWarps][F::kStages];
  __shared__ int s_last;
  __shared__ float* s_sums[F::kWarps];
  // What the tile loop has no use for, out of its registers: each warp's copy of
  // its part, the next one, and the share
  __shared__ Part s_now[F::kWarps], s_next[F::kWarps];
  __shared__ Share s_share[F::kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  const int G = a.Hq / a.Hkv;
  uint8_t* ring = smem + warp * F::kWarpBytes;
  uint8_t* factors = ring + F::kStages * F::kStageBytes;
  if (threadIdx.x == 0) tc::cta_abort_init();
  if (lane == 0)
    for (int i = 0; i < F::kStages; ++i) tc::mbar_init(&s_bar[warp][i], 1);
  tc::fence_mbar_init();

  // ---- this CTA's share of the work: every warp sums the sequences' units, 32
  // at a time, then finds the sequences that hold the share's ends
  auto sets_of = [&](const Seq& s) { return (s.rows * G + F::kVec - 1) / F::kVec; };
  auto units_of = [&](const Seq& s) {
    return s.rows * G > a.few ? 0u : unsigned(seq_units(s)) * a.Hkv * sets_of(s);
  };
  unsigned U = 0, pieces = 0;
  for (int i = lane; i < a.n_seq; i += 32) {
    const Seq s = sequence(a, i);
    const unsigned n = units_of(s);
    U += n;
    pieces += n ? a.Hkv * sets_of(s) : 0;
  }
  U = __reduce_add_sync(0xffffffffu, U);
  pieces = __reduce_add_sync(0xffffffffu, pieces);
  // counters of the kernel for many rows: 8 a CTA and one more
  if (a.many && warp == 0 && blockIdx.x < kCtas && lane < 9) a.counters[kItemCounter + blockIdx.x * 8 + lane] = 0u;
  if (U == 0) return;
  // One unit a warp at least.  A multiple of the pieces, if that leaves out no more
  // than a quarter of the CTAs: pieces of one length then begin where shares do, and
  // no CTA has two parts to join.  With / without: five rows over 8191 tokens 14.4/15.8
  // us, over 32768 27.8/31.6, 16 sequences of 4096 17.0/22.2 (with an eighth 22.3), 48
  // of 1500 18.4/24.0.  Ragged ones lose by it: 16 of 1640 to 4096 21.5/19.6, 48 of 600
  // to 1500 21.2/20.7, 160 drawn calls 13.36/13.29 in the geometric mean.
  unsigned ctas = min(gridDim.x, (U + F::kWarps - 1) / F::kWarps);
  if (ctas > pieces && ctas % pieces * 4 <= ctas) ctas -= ctas % pieces;
  if (blockIdx.x >= ctas) return;
  auto first_unit = [&](unsigned c) { return scaled(c, U, ctas, U); };
  // An end within kSnap tiles of an end of its piece moves there: what it would
  // split off costs less than the join.  A piece of up to 2 kSnap is never split.
  unsigned lo = first_unit(blockIdx.x), hi = first_unit(blockIdx.x + 1), seq_start = 0;
  int first_seq = 0;
  {
    unsigned before = 0, new_lo = lo, new_hi = hi;
    for (int i0 = 0; i0 < a.n_seq && before < hi; i0 += 32) {
      const int i = i0 + lane;
      const Seq s = i < a.n_seq ? sequence(a, i) : Seq{0, 0, 0};
      const unsigned n = units_of(s), each = seq_units(s);
      unsigned start = n;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const unsigned x = __shfl_up_sync(0xffffffffu, start, off);
        if (lane >= off) start += x;
      }
      const unsigned sum = __shfl_sync(0xffffffffu, start, 31);
      start += before - n;
      auto moved = [&](unsigned e) {
        const unsigned in = (e - start) % each, out = each - in;
        if (each > 2 * kSnap) return in <= kSnap ? e - in : (out <= kSnap ? e + out : e);
        return in < out ? e - in : e + out;
      };
      const unsigned has_lo = __ballot_sync(0xffffffffu, start <= lo && lo < start + n);
      const unsigned has_hi = __ballot_sync(0xffffffffu, start <= hi && hi < start + n);
      if (has_lo) {
        const int src = __ffs(has_lo) - 1;
        first_seq = i0 + src;
        seq_start = __shfl_sync(0xffffffffu, start, src);
        new_lo = __shfl_sync(0xffffffffu, lane == src ? moved(lo) : 0u, src);
      }
      if (has_hi) {
        const int src = __ffs(has_hi) - 1;
        new_hi = __shfl_sync(0xffffffffu, lane == src ? moved(hi) : 0u, src);
      }
      before += sum;
    }
    // the last end is U and lies in no sequence
    lo = new_lo;
    hi = new_hi;
  }
  if (lo >= hi) return;
  if (lane == 0) s_share[warp] = Share{hi, U, ctas};
  __syncthreads();  // the barriers are initialised
  auto cta_of = [&](unsigned u) {
    const Share h = s_share[warp];
    return scaled(u + 1, h.ctas, h.units, h.units, 1u);
  };

  // the part that holds unit u, of a sequence at or after p.seq (which starts at unit seq_start)
  auto part_at = [&](Part& p, unsigned u) {
    unsigned n = units_of(p.s);
    while (u >= seq_start + n) {
      seq_start += n;
      p.s = sequence(a, ++p.seq);
      n = units_of(p.s);
    }
    p.tiles = seq_tiles(p.s);
    const unsigned each = seq_units(p.s), hi = s_share[warp].hi;
    const int piece = int((u - seq_start) / each), sets = sets_of(p.s);
    p.g = piece / sets;
    p.v0 = (piece - p.g * sets) * F::kVec;
    p.start = seq_start + unsigned(piece) * each;
    p.next = min(hi, p.start + each);
    p.t_lo = int(u - p.start);
    p.t_hi = int(min(hi - p.start, unsigned(p.tiles)));
  };
  // tiles go to the warps in runs of up to kChunk
  auto run_of = [&](const Part& p) { return min(F::kChunk, (p.t_hi - p.t_lo + F::kWarps - 1) / F::kWarps); };
  // the part's end in tiles that hold tokens
  auto end_of = [&](const Part& p) { return min(p.t_hi, (p.s.len + kv4::kTile - 1) / kv4::kTile); };
  const int tpp = a.page / kv4::kTile;
  // page id of this lane's tile t of a run, loaded well before its copy; -1: none
  auto page_of = [&](const int* row, int run, int t, int end) {
    return lane < run && t < end ? __ldg(row + (a.tpp_shift >= 0 ? t >> a.tpp_shift : t / tpp)) : -1;
  };
  // bring a run's tiles (this lane's: t, on page id) of head g into a stage; whole warp
  auto fill = [&](int g, int run, int t, int end, int id, uint32_t stage) {
    uint64_t* bar = &s_bar[warp][stage];
    if (lane == 0)
      tc::mbar_expect_tx(bar, uint32_t(max(min(run, end - t), 0)) * kv4::tile_bytes(D));
    __syncwarp();
    if (lane < run && t < end) {
      if (unsigned(id) >= unsigned(a.num_pages)) {
        kv4::report(a.err, kv4::kErrPage);
        id = 0;
      }
      const int in = a.tpp_shift >= 0 ? t & (tpp - 1) : t % tpp;
      const uint64_t tile = (uint64_t(unsigned(id)) * unsigned(a.Hkv) + unsigned(g)) * unsigned(tpp) + unsigned(in);
      tc::bulk_load(ring + stage * F::kStageBytes + lane * kv4::tile_bytes(D),
                    a.pool + tile * kv4::tile_bytes(D), kv4::tile_bytes(D), bar);
    }
  };
  auto row_of = [&](const Part& p) { return a.table + p.seq * a.table_ld; };
  // the set's query rows as they are: lane (gid, tig) holds elements 8 tig .. of
  // each block of vector 8 j + gid
  auto load_q = [&](const Part& p, uint4 (&x)[kNT][nb]) {
#pragma unroll
    for (int j = 0; j < kNT; ++j) {
      const int v = p.v0 + 8 * j + gid;
#pragma unroll
      for (int b = 0; b < nb; ++b) x[j][b] = make_uint4(0u, 0u, 0u, 0u);
      if (v < p.s.rows * G) {
        const int r = v / G, h = v - r * G;
        const E* src = static_cast<const E*>(a.q) + (p.s.row0 + r) * a.q_row +
                       (p.g * G + h) * a.q_head + 8 * tig;
#pragma unroll
        for (int b = 0; b < nb; ++b) x[j][b] = q8(src + 32 * b, a.q_vec);
      }
    }
  };

  Part p;
  p.seq = first_seq;
  p.s = sequence(a, p.seq);
  part_at(p, lo);
  uint32_t it = 0;  // stages this warp has taken
  uint4 qx[kNT][nb];
  {
    const int run = run_of(p), t = p.t_lo + warp * run + lane, end = end_of(p);
    const int id = page_of(row_of(p), run, t, end);
    // the rows before the tiles: they would wait behind them
    load_q(p, qx);
    if (warp * run < p.t_hi - p.t_lo) fill(p.g, run, t, end, id, 0);
  }
  for (;;) {
    const int run = run_of(p), runs = (p.t_hi - p.t_lo + run - 1) / run, t_end = end_of(p);
    const int* row = row_of(p);
    const int g = p.g, len = p.s.len;
    int t0 = p.t_lo + warp * run;            // the warp's run,
    int t = t0 + F::kWarps * run + lane;     // this lane's tile of the next one to bring in
    int id = page_of(row, run, t, t_end);
    // the part after this one, and its first page
    int nid = -1;
    {
      Part np = p;
      if (p.next < s_share[warp].hi) {
        part_at(np, p.next);
        const int nrun = run_of(np);
        nid = page_of(row_of(np), nrun, np.t_lo + warp * nrun + lane, end_of(np));
      }
      __syncwarp();  // the copies of the part before are read
      if (lane == 0) {
        s_now[warp] = p;
        s_next[warp] = np;
      }
    }

    // ---- query rows to B fragments, scaled to a maximum near 2^15
    Query<D, kNT> q;
    q.all = len - p.s.rows + p.v0 / G + 1;
#pragma unroll
    for (int j = 0; j < kNT; ++j) {
      float2 x[nb][4];
      float am = 0.0f;
#pragma unroll
      for (int b = 0; b < nb; ++b) {
        x[b][0] = two_floats<E>(qx[j][b].x);
        x[b][1] = two_floats<E>(qx[j][b].y);
        x[b][2] = two_floats<E>(qx[j][b].z);
        x[b][3] = two_floats<E>(qx[j][b].w);
#pragma unroll
        for (int i = 0; i < 4; ++i) am = fmaxf(am, fmaxf(fabsf(x[b][i].x), fabsf(x[b][i].y)));
      }
      am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 1));
      am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 2));
      const int e = max(int(__float_as_uint(am) >> 23) - 127, -100);
      // the rows take the scale's sign; with a scale of zero all scores are zero
      float f = __uint_as_float(uint32_t(127 + 14 - e) << 23);
      f = a.scale == 0.0f ? 0.0f : copysignf(f, a.scale);
#pragma unroll
      for (int b = 0; b < nb; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          q.f[j][2 * b + (i >> 1)][i & 1] = pack_half(x[b][i].x * f, x[b][i].y * f);
      // back to the thread's score columns: vectors 2 tig and 2 tig + 1
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int ee = __shfl_sync(0xffffffffu, e, (2 * tig + i) * 4);
        q.qs[j][i] = fmaxf(fabsf(a.scale) * 1.44269504088896341f *
                               __uint_as_float(uint32_t(127 - 14 + 13 + ee) << 23), 1e-37f);
        const int c = p.v0 + 8 * j + 2 * tig + i;
        q.lim[j][i] = c < p.s.rows * G ? len - p.s.rows + c / G + 1 : 0;
      }
    }

    Running<D, kNT> w;
    w.top[0] = w.top[1] = 29u << 16 | 29u;  // blocks of zeros
#pragma unroll
    for (int j = 0; j < kNT; ++j) {
      w.m[j][0] = w.m[j][1] = -INFINITY;
      w.l[j][0] = w.l[j][1] = 0.0f;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) w.o[j][k][0] = w.o[j][k][1] = w.o[j][k][2] = w.o[j][k][3] = 0.0f;
    }
    for (int left = runs - warp; left > 0; left -= F::kWarps, ++it, t0 += F::kWarps * run) {
      if (left > F::kWarps) {  // the next one; this one is on its way
        __syncwarp();  // the stage's last readers are done
        fill(g, run, t, t_end, id, (it + 1) % F::kStages);
        t += F::kWarps * run;
        id = page_of(row, run, t, t_end);
      }
      tc::mbar_wait(&s_bar[warp][it % F::kStages], (it / F::kStages) & 1u, a.err, 1);
      const int n = min(run, t_end - t0);
      const uint8_t* stage = ring + (it % F::kStages) * F::kStageBytes;
      const int end = min(len, (t0 + n) * kv4::kTile);
      if (n > 1)
        attend_tiles<D, kNT, kPerSm, F::kChunk>(w, q, stage, factors, t0 * kv4::kTile, end);
      else if (n == 1)
        attend_tiles<D, kNT, kPerSm, 1>(w, q, stage, factors, t0 * kv4::kTile, end);
    }
    __syncwarp();
    p = s_now[warp];
    const Seq& s = p.s;
    const int nv = s.rows * G;
    const bool more_parts = p.next < s_share[warp].hi;
    // the next part's first tiles and rows are on their way during the join; the
    // sums take the place of the stage read last
    float* sums = reinterpret_cast<float*>(ring + ((it + 1) % F::kStages) * F::kStageBytes);
    if (more_parts) {
      const Part np = s_next[warp];
      const int nrun = run_of(np);
      load_q(np, qx);
      __syncwarp();
      if (warp * nrun < np.t_hi - np.t_lo)
        fill(np.g, nrun, np.t_lo + warp * nrun + lane, end_of(np), nid, it % F::kStages);
    }

    // ---- join the warps: sums of l over the quad's lanes, then through shared memory
    // the weights' 2^10 goes as well: values near the end of fp32 have no room for it
    float unit[nb];  // 2^(top_b - 127 - 15)
#pragma unroll
    for (int b = 0; b < nb; ++b) unit[b] = __uint_as_float((half_of(w.top[b % 2], b / 2) - 15) << 23);
#pragma unroll
    for (int j = 0; j < kNT; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int off = 4; off <= 16; off <<= 1)
          w.l[j][i] += __shfl_xor_sync(0xffffffffu, w.l[j][i], off);
        float* dst = sums + (8 * j + 2 * tig + i) * F::kAcc;
#pragma unroll
        for (int b = 0; b < nb; ++b)
          *reinterpret_cast<float4*>(dst + 32 * b + 4 * gid) =
              make_float4(w.o[j][2 * b][i] * unit[b], w.o[j][2 * b][i + 2] * unit[b],
                          w.o[j][2 * b + 1][i] * unit[b], w.o[j][2 * b + 1][i + 2] * unit[b]);
        if (gid == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(w.m[j][i], w.l[j][i] * 0x1p-10f);
      }
    if (lane == 0) s_sums[warp] = sums;
    __syncthreads();
    constexpr int kPer = D / 4, kRows = 32 / kPer;
    const int sub = lane / kPer, d0 = (lane % kPer) * 4;
    unsigned again = 0;  // this warp's vectors that are taken once more
    // vectors warp * kRows + sub, .. of the sums that the first `busy` warps left
    auto join_warps = [&](int busy, float* to) {
      for (int v = warp * kRows + sub; v < F::kVec; v += F::kWarps * kRows) {
        const float* src[F::kWarps];
        float2 ml[F::kWarps];
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < F::kWarps; ++i) src[i] = s_sums[i] + v * F::kAcc;
#pragma unroll
        for (int i = 0; i < F::kWarps; ++i) {
          ml[i] = i < busy ? *reinterpret_cast<const float2*>(src[i] + D) : make_float2(-INFINITY, 0.0f);
          m = fmaxf(m, ml[i].x);
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        float l = 0.0f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < F::kWarps; ++i) {
          if (i < busy && !out_of_range(ml[i].x)) {  // such sums are none: of no weight, or the vector is taken once more
            const float c = ex2(ml[i].x - ref);
            const float4 x = *reinterpret_cast<const float4*>(src[i] + d0);
            l = fmaf(c, ml[i].y, l);
            o[0] = fmaf(c, x.x, o[0]);
            o[1] = fmaf(c, x.y, o[1]);
            o[2] = fmaf(c, x.z, o[2]);
            o[3] = fmaf(c, x.w, o[3]);
          }
        }
        if (to) {
          *reinterpret_cast<float4*>(to + v * F::kAcc + d0) = make_float4(o[0], o[1], o[2], o[3]);
          if (d0 == 0) *reinterpret_cast<float2*>(to + v * F::kAcc + D) = make_float2(m, l);
        } else {
          const bool live = p.v0 + v < nv, redo = out_of_range(m);
          if (live && !redo) store_vector<E>(a, s, p.g, G, p.v0 + v, d0, o, l == 0.0f ? 0.0f : 1.0f / l, D);
          again |= __reduce_or_sync(0xffffffffu, live && redo ? 1u << v : 0u);
        }
      }
    };
    // A piece that several CTAs share is joined in two levels, by the last of a
    // group of its CTAs to arrive, then by the last of the groups; the order of
    // the sums does not depend on who arrives when.  One level for up to kOneLevel.
    int busy = min(F::kWarps, (p.t_hi - p.t_lo + run_of(p) - 1) / run_of(p));
    int c_first = 0, parts = 1, group = 1, first = 0, count = 1, stride = 1;
    if (p.t_lo != 0 || p.t_hi != p.tiles) {
      c_first = int(cta_of(p.start + kSnap));
      parts = int(cta_of(p.start + p.tiles - kSnap - 1)) - c_first + 1;
      group = parts <= kOneLevel ? parts : int(ceilf(sqrtf(float(parts))));
      first = (int(blockIdx.x) - c_first) / group * group;
      count = min(group, parts - first);
    }
    // the sums of the CTA that is the i-th of the piece, and of the group that begins there
    auto slot_at = [&](int i) { return slot_of<D, kNT, kPerSm>(a.part, c_first + i, i == 0); };
    float* to = parts == 1 ? nullptr : slot_of<D, kNT, kPerSm>(a.part, blockIdx.x, p.t_lo == 0);
    unsigned* counter = a.counters + 2 * (c_first + first) + (first == 0);
    for (int joined = 1;;) {  // CTAs of the piece whose sums this one has
      join_warps(busy, to);
      if (!to) break;
      __syncthreads();
      if (threadIdx.x == 0) {
        // release of the CTA's sums (ordered before by the barrier), acquire of the others'
        unsigned old;
        asm volatile("atom.acq_rel.gpu.global.inc.u32 %0, [%1], %2;"
                     : "=r"(old) : "l"(counter), "r"(unsigned(count - 1)) : "memory");
        s_last = old == unsigned(count - 1);
      }
      __syncthreads();
      if (!s_last) break;
      constexpr int kN = F::kVec / kRows;
      float m[kN], l[kN];
      float4 o[kN];
      join_rows<D, kNT, kPerSm>(warp, F::kWarps, count, [&](int i) { return slot_at(first + i * stride); }, m, l, o);
#pragma unroll
      for (int k = 0; k < kN; ++k) {
        float* dst = sums + (k * kRows + sub) * F::kAcc;
        *reinterpret_cast<float4*>(dst + d0) = o[k];
        if (d0 == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(m[k], l[k]);
      }
      __syncthreads();
      busy = min(F::kWarps, count);
      joined *= group;
      to = joined >= parts ? nullptr : slot_at(first);
      first = 0;
      stride = group;
      count = (parts + group - 1) / group;
      counter = a.counters + 2 * kFewCtas + c_first;
    }
    for (; again; again &= again - 1) {
      const int v = s_now[warp].v0 + __ffs(again) - 1;
      const Seq& x = s_now[warp].s;
      attend_exactly<E, D>(a, s_now[warp].seq, x.row0 + v / G, s_now[warp].g * G + v % G,
                           x.len - x.rows + v / G + 1);
    }
    if (!more_parts) break;
    // the sums are read: their memory, written by ordinary stores, takes tiles
    // from bulk copies again
    tc::fence_proxy_async_smem();
    __syncthreads();
    p = s_next[warp];
  }
  if (tc::cta_aborted()) tc::drain_ring(s_bar[warp], F::kStages, it);
}

template <class E, int D, int kNT, int kPerSm>
cudaError_t launch_few(const AttnArgs& a, cudaStream_t s) {
  using F = Few<D, kNT, kPerSm>;
  const void* fn = reinterpret_cast<const void*>(kv4_attn_few_kernel<E, D, kNT, kPerSm>);
  const cudaError_t e = ensure_dynamic_smem(fn, F::kSmem);
  if (e != cudaSuccess) return e;
  kv4_attn_few_kernel<E, D, kNT, kPerSm><<<kSms * kPerSm, F::kThreads, F::kSmem, s>>>(a);
  return cudaGetLastError();
}

// Vectors of a set: 8, or 16 (a KV head's bytes are then read and decoded half as
// often, at 255 registers and some spills) where the call has more than 24 sets of 8.
// 8 / 16, us, for 256, 1024, 4096, 16384, 65536 tokens:
//    8 sets (4 pairs, 16 vectors)   8.4/10.1  10.6/13.2  13.1/19.0  16.1/19.9  26.1/25.5
//   20      (4, 40)                 8.7/10.6  10.9/13.5  12.6/17.1  19.4/20.9  44.3/44.2
//   32      (4, 64)                 8.8/10.7  10.9/13.6  13.6/17.1  24.8/23.9  68.4/54.4
//   32      (16, 16)                8.8/10.6  10.9/13.5  13.5/17.3  24.8/23.7  69.4/55.4
//   64      (32, 16)                8.9/10.7  11.0/13.7  17.0/17.1  39.1/34.6
int set_vectors(long long n_seq, int Hkv, long long vectors) {
  return n_seq * Hkv * ((std::min(vectors, (long long)kFew) + 7) / 8) <= 24 || vectors <= 8 ? 8 : 16;
}

// One large CTA an SM for up to 64 pairs of a sequence and KV head (fewer sums to
// join), three (two with 16 vectors) small ones for more (one's start and join hide
// behind the others).  Large / small, us, 8 query heads a KV head, D 128:
//   pairs                 4         32        64        128       256
//   1024 tokens each      10.4/12.1 10.9/12.6 11.0/14.4 11.0/14.2 19.2/18.1
//   4096                  14.5/16.2 13.7/16.6 17.1/18.1 22.4/25.3 48.6/43.3
//   103 .. 4096           11.6/13.9 13.7/17.8 18.3/17.4 29.1/21.0 44.6/28.0
//   two rows each, 4096   19.1/22.9 17.2/22.8 22.9/22.9 31.2/33.8 66.0/53.7
// (pairs of up to 256 tokens gain 1 us from small CTAs at any count.)
// Sequences of more than kFew vectors go to the kernel for many rows, which reads a
// tile for 256 vectors at once.  Few / many, us, 4096 tokens: one sequence 17.2/35.9
// with 64 vectors a KV head, 17.1/37.0 with 128; 16 sequences 54.2/56.6 with 48,
// 63.9/57.3 with 64, 74.7/57.6 with 80.
template <class E, int D>
cudaError_t launch(AttnArgs& a, cudaStream_t s) {
  const long long vectors = (long long)a.max_q * (a.Hq / a.Hkv);
  const bool many_pieces = (long long)a.n_seq * a.Hkv > 64;
  a.few = kFew;
  a.many = vectors > kFew;
  cudaError_t e;
  if (set_vectors(a.n_seq, a.Hkv, vectors) == 8)
    e = many_pieces ? launch_few<E, D, 1, 3>(a, s) : launch_few<E, D, 1, 1>(a, s);
  else
    e = many_pieces ? launch_few<E, D, 2, 2>(a, s) : launch_few<E, D, 2, 1>(a, s);
  if (e == cudaSuccess && a.many)
    e = launch_kv4_prefill(a, std::is_same<E, __nv_bfloat16>::value, D, s);
  return e;
}

}  // namespace
}  // namespace mfi

extern "C" size_t mfi_kv4_attn_workspace_bytes(int n_seq, int Hq, int Hkv, int D, int max_q) {
  if (n_seq <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || (D != 64 && D != 128) || max_q <= 0)
    return 0;
  const bool many = (long long)max_q * (Hq / Hkv) > mfi::kv4::kFew;
  return mfi::kv4::kCounterBytes + (many ? mfi::kv4::many_bytes(D) : mfi::kv4::few_bytes(D));
}

extern "C" int mfi_kv4_attn_init_workspace(void* workspace, size_t workspace_bytes, void* stream) {
  if (!workspace) return mfi::set_last_error(MFI_ERR_ARG, "null pointer");
  const cudaError_t e = cudaMemsetAsync(workspace, 0, workspace_bytes,
                                        reinterpret_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? MFI_OK : mfi::set_last_error(MFI_ERR_CUDA, cudaGetErrorString(e));
}

extern "C" int mfi_kv4_attn(const void* q, int dtype, long long q_row, long long q_head,
                            const uint8_t* pool, const int32_t* table, long long table_ld,
                            const int32_t* kv_lens, const int32_t* cu_q, void* out, int T,
                            int max_q, int n_seq, int Hq, int Hkv, int D, int page, int num_pages,
                            int width, float scale, void* workspace, size_t workspace_bytes,
                            void* stream) {
  if (dtype != MFI_F16 && dtype != MFI_BF16)
    return mfi::set_last_error(MFI_ERR_ARG, "kv4_attn: q must be MFI_F16 or MFI_BF16");
  const int rc = mfi::kv4_check_pool(pool, Hkv, D, page, num_pages);
  if (rc != MFI_OK) return rc;
  if (T < 0 || max_q < 0 || n_seq < 0 || width < 0)
    return mfi::set_last_error(MFI_ERR_ARG, "kv4_attn: T, max_q, n_seq and width must not be negative");
  if (Hq <= 0 || Hq % Hkv != 0)
    return mfi::set_last_error(MFI_ERR_ARG, "kv4_attn: Hq must be a positive multiple of Hkv");
  if (!cu_q && (long long)n_seq * max_q != T)
    return mfi::set_last_error(MFI_ERR_ARG, "kv4_attn: without cu_q there are n_seq * max_q rows");
  if (T == 0 || n_seq == 0 || max_q == 0) return MFI_OK;
  if (!q || (!table && width > 0) || !kv_lens || !out || !workspace)
    return mfi::set_last_error(MFI_ERR_ARG, "null pointer");
  if (reinterpret_cast<uintptr_t>(out) & 15)
    return mfi::set_last_error(MFI_ERR_ARG, "kv4_attn: out must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(workspace) & 255)
    return mfi::set_last_error(MFI_ERR_ARG, "kv4_attn: the workspace must be 256-byte aligned");
  if (workspace_bytes < mfi_kv4_attn_workspace_bytes(n_seq, Hq, Hkv, D, max_q))
    return mfi::set_last_error(MFI_ERR_WORKSPACE, "workspace smaller than the kv4_attn workspace query");
  // units of work of the kernel for few rows (a tile of a KV head for a set of
  // vectors) are counted in 31 bits: as many as the table has room for, and sets as
  // the rows allow.  The items of the other one are fewer than the rows of `out`.
  const double vectors = fmin(double(max_q) * (Hq / Hkv), double(mfi::kv4::kFew));
  const double per = mfi::set_vectors(n_seq, Hkv, (long long)max_q * (Hq / Hkv));
  const double sets = fmin(n_seq * ceil(vectors / per), n_seq + double(T) * (Hq / Hkv) / per);
  const double tiles = fmax(ceil(double(width) * page / mfi::kv4::kTile), mfi::kLeast);
  if (sets * Hkv * tiles >= 2147483648.0)
    return mfi::set_last_error(MFI_ERR_ARG, "kv4_attn: more than 2^31 tiles of work in one call");
  mfi::kv4::AttnArgs a{};
  a.q = q; a.q_row = q_row; a.q_head = q_head;
  a.pool = pool; a.table = table; a.table_ld = table_ld;
  a.kv_lens = kv_lens; a.cu_q = cu_q; a.out = out;
  a.err = mfi::device_error_flag();
  a.T = T; a.max_q = max_q; a.n_seq = n_seq; a.Hq = Hq; a.Hkv = Hkv;
  a.page = page; a.num_pages = num_pages; a.width = width;
  a.scale = scale;
  const int tpp = page / mfi::kv4::kTile;
  a.q_vec = !((reinterpret_cast<uintptr_t>(q) | uintptr_t(q_row * 2) | uintptr_t(q_head * 2)) & 15);
  a.tpp_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (tpp == 1 << i) a.tpp_shift = i;
  a.counters = static_cast<unsigned*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + mfi::kv4::kCounterBytes);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (dtype == MFI_BF16)
    e = D == 128 ? mfi::launch<__nv_bfloat16, 128>(a, s) : mfi::launch<__nv_bfloat16, 64>(a, s);
  else
    e = D == 128 ? mfi::launch<__half, 128>(a, s) : mfi::launch<__half, 64>(a, s);
  return e == cudaSuccess ? MFI_OK : mfi::set_last_error(MFI_ERR_CUDA, cudaGetErrorString(e));
}
