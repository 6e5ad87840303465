// kv4_prefill.cu — attention over the paged 4-bit KV cache for many rows
// (prompts and their chunks) on the tcgen05 tensor cores.  Semantics and
// arguments: kv4_attn.cu; layout: kv4.cuh.
//
// A vector is one row of one query head; an item is 256 vectors (two tiles of
// 128) of a sequence and KV head, against the tokens that the last of them sees,
// 64 a step.  One persistent CTA per SM takes items from a counter, the longest
// of a sequence first.  With fewer items than CTAs the tokens of each are split
// into parts, whose sums the last part's warps join.  A CTA's roles:
//   warp 13      finds the next item, brings the tokens' tiles in by bulk copies
//   warp 15      finds the largest codes of a step
//   warps 8-11   decode its tiles to fp16 operands in shared memory (128-byte swizzle)
//   warps 12, 14 issue S_i = Q_i K^T of step s + 2 and O_i += P_i V of step s, one
//                warp a tile i: while one waits the other's products run
//   warps 0-7    softmax, one thread a vector: S from TMEM, P as fp16 back into
//                its place, O rescaled in TMEM when the maximum has moved, O out
// TMEM: of each tile two S of 64 columns (P in the first half of its S), then O_0
// and O_1.  Two S a tile keep the softmax supplied while the tensor cores are at
// the step before; with one S of 128 tokens a tile its warps and the tensor cores
// waited for each other (16384 rows: 1.98 ms, now 1.67), although a product of 64 columns
// takes 50 clocks and one of 128 takes 65 (both operands from shared memory).
//
// The operands are fp16: a query row times a power of two that brings its
// maximum to [2^14, 2^15), a key or value element times 2^(c - ref + 13).  The
// keys' ref is the largest code of the 64 tokens: exact unless 2^-37 below it.  The
// values have one for each block of 32 channels, which O refers to as well: set 3
// above the block's largest code, and again when a code passes it, so exact unless
// 2^-34 below the largest so far of the same block.  The few rows that lose by it (they
// do not see the strong values, or their scores are huge) are taken once more in fp32.
// P is rounded to fp16 after a factor 2^6; the maximum that it refers to moves
// when it is passed by 2^9 (2^7: 3% more for a prompt of 16384 tokens), so P stays below 2^15;
// weights below 2^-20 of the reference lose bits, those below 2^-31 vanish.  l and O
// are fp32.
#include <cuda_fp16.h>

#include <atomic>

#include "../../include/moe_fp4.h"
#include "kv4_attn.cuh"
#include "tc_ptx.cuh"
#include "tmap.cuh"
#include "work.cuh"

namespace mfi {
namespace {

using namespace kv4;

constexpr int kTok = 64;                   // tokens of a step
constexpr int kSlots = 4;                  // steps on their way
constexpr int kRows = 128;                 // vectors of a tile
constexpr int kThreads = 512;
constexpr int kRegsSoftmax = 168, kRegsDecode = 112, kRegsOther = 64;
static_assert(2 * kRegsSoftmax + kRegsDecode + kRegsOther <= 512, "registers of the launch: 128 a thread");
constexpr float kLazy = 9.0f, kShift = 6.0f;  // log2: the maximum's slack, the weights' factor
constexpr uint32_t kVSlack = 3;               // log2: the value references' slack
constexpr int kUp = 13;                       // log2: the elements' factor

template <int D>
struct Many {
  static constexpr int kQ = kRows * D * 2;                   // a tile's query rows
  static constexpr int kOperand = kTok * D * 2;              // K or V of a step
  static constexpr int kRaw = kTok / kTile * tile_bytes(D);  // a step's tiles
  static constexpr int kOffK = 2 * kQ, kOffV = kOffK + kSlots * kOperand;
  static constexpr int kOffRaw = kOffV + kSlots * kOperand;
  static constexpr int kSmem = kOffRaw + kSlots * kRaw;
};

struct Item {
  int valid, seq, row0, rows, len, g, v0;
  int step0, steps;         // of this part
  int part, parts, index;   // the part's index among all parts of the call
};

// Parts of an item: no more than the CTAs allow, of at least kMinSteps steps (a
// part starts in about 5 us, 8 steps take about as long), at most kMaxParts (they
// are joined by one CTA's warps).  kMinSteps 4, 8, 16: 100 rows over 2048 tokens, 4
// KV heads of 8, 40.0, 40.1, 50.4 us, over 1024 33.8, 32.6, 32.8; kMaxParts 6, 12,
// 18: 100 rows over 8192, one KV head, 51.5, 47.4, 53.2, 40 over 32768 114, 81, 75.
constexpr int kMinSteps = 8, kMaxParts = 12;

// An operand of R rows: halves of 64 elements, each R rows of 128 bytes in the
// 128-byte swizzle.  Byte offset of 16-byte chunk c (8 elements) of row r:
template <int R>
__device__ __forceinline__ uint32_t operand_at(int r, int c) {
  return uint32_t(c >> 3) * (R * 128) + uint32_t(r) * 128 + (uint32_t((c & 7) ^ (r & 7)) << 4);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(add))
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(uint32_t(add))
      : "memory");
}
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// (a.x, a.y) * b + c, each half on its own
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n"
      " fma.rn.f32x2 x, x, y, z;\n mov.b64 {%0, %1}, x;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n"
      " add.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}

struct Bars {
  uint64_t item_full[2], item_empty[2];            // the next item's description
  uint64_t raw_full[kSlots], raw_empty[kSlots];    // a step's tiles,
  uint64_t ref_full[kSlots];                       // its codes' references,
  uint64_t kv_full[kSlots], kv_empty[kSlots];      // its operands
  uint64_t q_full[2];                              // of tile i: query rows written,
  uint64_t s_full[2][2], p_full[2][2];             // scores there, weights there (by step & 1),
  uint64_t o_done[2][2];                           // products added (by step & 1)
  uint64_t drain[2];
};

template <class E, int D>
__global__ void __launch_bounds__(kThreads, 1) kv4_attn_many_kernel(AttnArgs a) {
  using M = Many<D>;
  constexpr int nb = D / 32;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ Bars bar;
  __shared__ Item s_item[2];
  __shared__ int s_nan[2][4];     // of an item: first token whose value block is NaN,
  __shared__ int s_far[2];        // values far stronger than others that some rows see without them
  // of a step: the key code that its operands refer to, whether there are NaN values
  // (bit 0) and whether the values' codes are others than the step's before (bit 1),
  // these, of blocks 0 and 2 (halves), 1 and 3.  Its writer is at most 2 kSlots steps
  // ahead of its last reader.
  __shared__ uint4 s_ref[4 * kSlots];
  __shared__ uint32_t s_tmem;
  // (from lane 0: the roles' branches are then known to be uniform)
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int G = a.Hq / a.Hkv;

  if (threadIdx.x == 0) {
    tc::cta_abort_init();
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&bar.item_full[i], 1);
      tc::mbar_init(&bar.item_empty[i], 8 + 4 + 1 + 64);  // a lane of each warp that reads it, all of warps 12 and 14
      tc::mbar_init(&bar.drain[i], 1);
      tc::mbar_init(&bar.q_full[i], 4);
      for (int b = 0; b < 2; ++b) {
        tc::mbar_init(&bar.s_full[i][b], 1);
        tc::mbar_init(&bar.p_full[i][b], 4);
        tc::mbar_init(&bar.o_done[i][b], 1);
      }
    }
    for (int i = 0; i < kSlots; ++i) {
      tc::mbar_init(&bar.raw_full[i], 1);
      tc::mbar_init(&bar.raw_empty[i], 4);
      tc::mbar_init(&bar.ref_full[i], 1);
      tc::mbar_init(&bar.kv_full[i], 4);
      tc::mbar_init(&bar.kv_empty[i], 2);
    }
    tc::fence_mbar_init();
  }
  if (warp == 12) tc::tmem_alloc(&s_tmem, 512);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
  int* err = a.err;

  // wait for the n-th completion (from 0) of a barrier; the warp goes on or gives
  // up as one
  auto wait = [&](uint64_t* b, uint32_t n, int code) {
    return tc::mbar_wait_warp(b, n & 1u, err, code);
  };
  // the n-th completion of the barrier of step n's slot
  auto wait_slot = [&](uint64_t* b, uint32_t n, int code) { return wait(b + n % kSlots, n / kSlots, code); };

  if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (warp == 13) {
      // ---- items and their tiles
      const int tpp = a.page / kTile;
      const uint64_t page_bytes = uint64_t(a.Hkv) * tpp * tile_bytes(D);
      uint32_t step = 0, filled = 0;
      auto items_of = [&](const Seq& s) {
        return s.rows * G > a.few ? unsigned((s.rows * G + 2 * kRows - 1) / (2 * kRows)) * a.Hkv : 0u;
      };
      unsigned all_items = 0;
      for (int i = lane; i < a.n_seq; i += 32) all_items += items_of(sequence(a, i));
      all_items = __reduce_add_sync(0xffffffffu, all_items);
      const int most = all_items ? min(kMaxParts, int(gridDim.x / all_items)) : 0;
      // the same for all items of a sequence; none is left without a step: the item
      // of the first rows sees len - rows + 1 tokens at least
      auto parts_of = [&](const Seq& s) {
        const int few_steps = (s.len - s.rows) / kTok;
        return unsigned(max(1, min(most, few_steps / kMinSteps)));
      };
      for (uint32_t n = 0;; ++n) {
        unsigned idx = 0;
        if (lane == 0) idx = atomicAdd(a.counters + kItemCounter, 1u);
        idx = __shfl_sync(0xffffffffu, idx, 0);
        Item it{};
        unsigned before = 0;
        for (int i0 = 0; i0 < a.n_seq; i0 += 32) {
          const int i = i0 + lane;
          const Seq s = i < a.n_seq ? sequence(a, i) : Seq{0, 0, 0};
          const unsigned parts = parts_of(s), items = items_of(s) * parts;
          unsigned start = items;
#pragma unroll
          for (int off = 1; off < 32; off <<= 1) {
            const unsigned x = __shfl_up_sync(0xffffffffu, start, off);
            if (lane >= off) start += x;
          }
          const unsigned sum = __shfl_sync(0xffffffffu, start, 31);
          start += before - items;
          const unsigned has = __ballot_sync(0xffffffffu, start <= idx && idx < start + items);
          if (has) {
            const int src = __ffs(has) - 1;
            it.valid = 1;
            it.seq = i0 + src;
            it.row0 = __shfl_sync(0xffffffffu, s.row0, src);
            it.rows = __shfl_sync(0xffffffffu, s.rows, src);
            it.len = __shfl_sync(0xffffffffu, s.len, src);
            it.parts = int(__shfl_sync(0xffffffffu, parts, src));
            const unsigned all = __shfl_sync(0xffffffffu, items, src) / it.parts;
            const unsigned in = idx - __shfl_sync(0xffffffffu, start, src);
            it.part = int(in % it.parts);
            it.index = int(idx);
            const unsigned item = in / it.parts;
            it.g = int(item % a.Hkv);
            it.v0 = int(all / a.Hkv - 1 - item / a.Hkv) * 2 * kRows;  // the rows that see most first
            const int last = min(it.v0 + 2 * kRows, it.rows * G) - 1;
            const int steps = max(1, (it.len - it.rows + last / G + 1 + kTok - 1) / kTok);
            it.step0 = int((long long)steps * it.part / it.parts);
            it.steps = int((long long)steps * (it.part + 1) / it.parts) - it.step0;
            break;
          }
          before += sum;
        }
        const uint32_t slot = n & 1u;
        if (n >= 2 && !wait(&bar.item_empty[slot], (n >> 1) - 1, 1)) break;
        if (lane == 0) {
          s_item[slot] = it;
          for (int b = 0; b < 4; ++b) s_nan[slot][b] = 0x7FFFFFFF;
          s_far[slot] = 0;
          tc::mbar_arrive(&bar.item_full[slot]);
        }
        if (!it.valid) break;
        const int have = (it.len + kTile - 1) / kTile;
        const int* row = a.table + it.seq * a.table_ld;
        auto page_of = [&](int t) {
          return lane < kTok / kTile && t < have ? __ldg(row + (a.tpp_shift >= 0 ? t >> a.tpp_shift : t / tpp))
                                                 : -1;
        };
        int t = it.step0 * (kTok / kTile) + lane, id = page_of(t);
        bool ok = true;
        for (int j = 0; j < it.steps; ++j, ++step) {
          const uint32_t st = step % kSlots;
          ok = step < kSlots || wait_slot(bar.raw_empty, step - kSlots, 1);
          if (!ok) break;
          if (lane == 0)
            tc::mbar_expect_tx(&bar.raw_full[st],
                               uint32_t(max(min(kTok / kTile, have - t), 0)) * tile_bytes(D));
          __syncwarp();
          filled = step + 1;
          if (lane < kTok / kTile && t < have) {
            if (unsigned(id) >= unsigned(a.num_pages)) {
              report(err, kErrPage);
              id = 0;
            }
            const int in = it.g * tpp + (a.tpp_shift >= 0 ? t & (tpp - 1) : t % tpp);
            tc::bulk_load(smem + M::kOffRaw + st * M::kRaw + lane * tile_bytes(D),
                          a.pool + unsigned(id) * page_bytes + uint64_t(unsigned(in)) * tile_bytes(D),
                          tile_bytes(D), &bar.raw_full[st]);
          }
          t += kTok / kTile;
          id = page_of(t);
        }
        if (!ok) break;
      }
      if (tc::cta_aborted()) tc::drain_ring(bar.raw_full, kSlots, filled);
    } else if (warp == 12 || warp == 14) {
      // ---- MMA issue of tile i: the whole warp goes along, so that the descriptors stay in
      // uniform registers, one lane issues.  Descriptors are advanced by adding to
      // their address field (bytes / 16).
      constexpr uint32_t kIdesc = (1u << 4) | (uint32_t(kTok >> 3) << 17) | (uint32_t(kRows >> 4) << 24);
      constexpr uint32_t kIdescPV =  // B (values) with the elements along N contiguous
          (1u << 4) | (1u << 16) | (uint32_t(D >> 3) << 17) | (uint32_t(kRows >> 4) << 24);
      const uint32_t base = tc::smem_u32(smem);
      const uint64_t dq = tc::make_sdesc(base, 16, 1024, tc::kLayoutSW128);
      const uint64_t dk = tc::make_sdesc(base + M::kOffK, 16, 1024, tc::kLayoutSW128);
      const uint64_t dv = tc::make_sdesc(base + M::kOffV, kTok * 128, 1024, tc::kLayoutSW128);
      const int i = (warp - 12) >> 1;
      const bool leader = tc::elect_one();
      auto commit = [&](uint64_t* b) {
        if (leader) tc::tc_commit(b);
      };
      auto scores = [&](uint32_t g) {  // of step g
        tc::tc_fence_after();
        const uint64_t q = dq + uint32_t(i) * (M::kQ >> 4), k = dk + (g % kSlots) * (M::kOperand >> 4);
        const uint32_t d = tmem + i * 128 + (g & 1u) * 64;
        if (leader) {
#pragma unroll
          for (int x = 0; x < D / 16; ++x)
            mma_ss(d, q + (((x >> 2) * (kRows * 128) + (x & 3) * 32) >> 4),
                   k + (((x >> 2) * (kTok * 128) + (x & 3) * 32) >> 4), kIdesc, x != 0);
          tc::tc_commit(&bar.s_full[i][g & 1u]);
        }
      };
      auto values = [&](uint32_t g, bool add) {
        tc::tc_fence_after();
        const uint64_t v = dv + (g % kSlots) * (M::kOperand >> 4);
        const uint32_t p = tmem + i * 128 + (g & 1u) * 64;
        if (leader) {
#pragma unroll
          for (int x = 0; x < kTok / 16; ++x)
            mma_ts(tmem + 256 + i * 128, p + x * 8, v + x * (2048 >> 4), kIdescPV, add || x != 0);
          tc::tc_commit(&bar.o_done[i][g & 1u]);
        }
      };
      uint32_t g = 0;  // steps of all items
      bool ok = true;
      for (uint32_t n = 0; ok; ++n) {
        const uint32_t slot = n & 1u;
        if (!wait(&bar.item_full[slot], n >> 1, 2)) break;
        const int valid = __shfl_sync(0xffffffffu, s_item[slot].valid, 0);
        const int steps = __shfl_sync(0xffffffffu, s_item[slot].steps, 0);
        tc::mbar_arrive(&bar.item_empty[slot]);
        if (!valid) break;
        ok = wait(&bar.q_full[i], n, 2);
        // the scores run two steps ahead of the products
        for (int j = 0; j < 2 && j < steps && ok; ++j) {
          ok = wait_slot(bar.kv_full, g + j, 2);
          if (!ok) break;
          scores(g + j);
        }
        for (int j = 0; j < steps && ok; ++j, ++g) {
          const bool more = j + 2 < steps;
          ok = wait(&bar.p_full[i][g & 1u], g >> 1, 2);
          if (!ok) break;
          values(g, j != 0);
          commit(&bar.kv_empty[g % kSlots]);  // of its keys too: their scores came before
          if (more) {
            ok = wait_slot(bar.kv_full, g + 2, 2);
            if (!ok) break;
            scores(g + 2);
          }
        }
      }
      if (tc::cta_aborted() && leader) tc::drain_mma(&bar.drain[i]);
    } else if (warp == 15) {
      // ---- the codes that the operands refer to (255, NaN, not counted)
      uint32_t step = 0;
      bool ok = true;
      for (uint32_t n = 0; ok; ++n) {
        const uint32_t slot = n & 1u;
        if (!wait(&bar.item_full[slot], n >> 1, 1)) break;
        const int valid = s_item[slot].valid, steps = s_item[slot].steps;
        const int pos = s_item[slot].step0 * kTok, len = s_item[slot].len - pos;  // of the part
        const int all = len - s_item[slot].rows + s_item[slot].v0 / G + 1;  // tokens that all rows see
        uint32_t v02 = 28u << 16 | 28u, v13 = v02;  // blocks of zeros
        for (int j = 0; valid && j < steps; ++j, ++step) {
          ok = wait_slot(bar.raw_full, step, 1);
          if (!ok) break;
          const uint8_t* raw = smem + M::kOffRaw + (step % kSlots) * M::kRaw;
          uint32_t wk[kTok / 32], wv[kTok / 32];  // codes of tokens lane, lane + 32
#pragma unroll
          for (int x = 0; x < kTok / 32; ++x) {
            const int tok = x * 32 + lane;
            const uint8_t* c = raw + (tok / kTile) * tile_bytes(D) + 16 * D + (tok % kTile) * nb;
            wk[x] = nb == 4 ? *reinterpret_cast<const uint32_t*>(c) : *reinterpret_cast<const uint16_t*>(c);
            c += D / 2;
            wv[x] = nb == 4 ? *reinterpret_cast<const uint32_t*>(c) : *reinterpret_cast<const uint16_t*>(c);
            if (j * kTok + tok >= len) wk[x] = wv[x] = 0u;
          }
          auto evens = [](const uint32_t (&w)[kTok / 32]) { return __vmaxu2(w[0] & 0x00FF00FFu, w[1] & 0x00FF00FFu); };
          auto odds = [](const uint32_t (&w)[kTok / 32]) {
            return __vmaxu2((w[0] >> 8) & 0x00FF00FFu, (w[1] >> 8) & 0x00FF00FFu);
          };
          static_assert(kTok == 64, "two tokens a lane");
          auto largest = [&] {
            const uint32_t m = __vmaxu2(evens(wk), odds(wk));
            return __reduce_max_sync(0xffffffffu, max(m & 0xFFFFu, m >> 16));
          };
          uint32_t kref = largest();
          if (kref == 255u) {  // rare: once more without them
#pragma unroll
            for (int x = 0; x < kTok / 32; ++x) wk[x] &= ~__vcmpeq4(wk[x], 0xFFFFFFFFu);
            kref = largest();
          }
          kref = max(kref, 28u);
          // the values' references, of 254 at most, move when a code passes one
          uint32_t e = __vmaxu2(evens(wv), v02), o = __vmaxu2(odds(wv), v13), nan = 0u, moved = 0u;
          if (__any_sync(0xffffffffu, e != v02 || o != v13)) {
#pragma unroll
            for (int x = 0; x < kTok / 32; ++x) {
              const uint32_t bad = __vcmpeq4(wv[x], 0xFFFFFFFFu);
              // a NaN value block counts for the rows that see it only: noted here,
              // written at the end, and zero in the product
              for (int b = 0; b < nb; ++b)
                if ((bad >> (8 * b)) & 1u) atomicMin(&s_nan[slot][b], pos + j * kTok + x * 32 + lane);
              wv[x] &= ~bad;
              nan |= bad;
            }
            nan = __any_sync(0xffffffffu, nan != 0u);
            e = __vmaxu2(evens(wv), v02);
            o = __vmaxu2(odds(wv), v13);
            auto passed = [&](uint32_t now, uint32_t then) {
              const uint32_t top = __reduce_max_sync(0xffffffffu, now);
              return top > then ? min(top + kVSlack, 254u) : then;
            };
            const uint32_t n02 = passed(e & 0xFFFFu, v02 & 0xFFFFu) | passed(e >> 16, v02 >> 16) << 16;
            const uint32_t n13 = passed(o & 0xFFFFu, v13 & 0xFFFFu) | passed(o >> 16, v13 >> 16) << 16;
            moved = j > 0 && (n02 != v02 || n13 != v13) ? 2u : 0u;
            if ((j + 1) * kTok > all) {
              bool far = false;
#pragma unroll
              for (int b = 0; b < nb; ++b) {
                const uint32_t then = half_of(b % 2 ? v13 : v02, b / 2), now = half_of(b % 2 ? n13 : n02, b / 2);
                uint32_t lo = then > 28u ? then - kVSlack : 255u;
#pragma unroll
                for (int x = 0; x < kTok / 32; ++x) {
                  const uint32_t c = (wv[x] >> (8 * b)) & 0xFFu;
                  if (c > 28u) lo = min(lo, c);
                }
                far |= now > then && int(now) - int(__reduce_min_sync(0xffffffffu, lo)) > 28 + int(kVSlack);
              }
              if (far && lane == 0) s_far[slot] = 1;
            }
            v02 = n02;
            v13 = n13;
          }
          __syncwarp();
          if (lane == 0) {
            s_ref[step % (4 * kSlots)] = make_uint4(kref, nan | moved, v02, v13);
            tc::mbar_arrive(&bar.ref_full[step % kSlots]);
          }
        }
        if (lane == 0) tc::mbar_arrive(&bar.item_empty[slot]);
        if (!valid) break;
      }
    }
  } else if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsDecode));
    // ---- decode: a warp a tile; lane (row, quarter t of the row) of 8 rows at a
    // time, rows r and r + 4 side by side: their swizzled chunks share no banks
    constexpr int kMine = kTok / 4;
    static_assert(kMine == kTile, "a tile a warp");
    const int dw = warp - 8, t = lane & 3, r8 = ((lane >> 2) & 1) * 4 + (lane >> 3);
    const int at = (dw * kMine + r8) * 128 + ((t ^ r8) << 4);  // of the row's chunk t
    uint32_t step = 0;
    for (uint32_t n = 0;; ++n) {
      const uint32_t slot = n & 1u;
      if (!wait(&bar.item_full[slot], n >> 1, 1)) break;
      const int steps = s_item[slot].steps, valid = s_item[slot].valid;
      const int len = s_item[slot].len - s_item[slot].step0 * kTok;  // of the part on
      bool ok = true;
      for (int j = 0; valid && j < steps; ++j, ++step) {
        const uint32_t st = step % kSlots;
        ok = wait(&bar.ref_full[st], step / kSlots, 1);
        if (!ok) break;
        const uint4 ref = s_ref[step % (4 * kSlots)];
        const uint8_t* tile = smem + M::kOffRaw + st * M::kRaw + dw * tile_bytes(D);
        uint32_t w[2][2][nb], cw[2][2];  // of key and value rows r8, r8 + 8
#pragma unroll
        for (int kv = 0; kv < 2; ++kv)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int in = x * 8 + r8;
            const uint8_t* c = tile + 16 * D + kv * (D / 2) + in * nb;
            cw[kv][x] = nb == 4 ? *reinterpret_cast<const uint32_t*>(c) : *reinterpret_cast<const uint16_t*>(c);
            if (j * kTok + dw * kMine + in >= len) cw[kv][x] = 0;
            const uint8_t* src = tile + kv * 8 * D + in * (D / 2) + t * (4 * nb);
            if (nb == 4) {
              const uint4 y = *reinterpret_cast<const uint4*>(src);
              w[kv][x][0] = y.x; w[kv][x][1] = y.y; w[kv][x][nb - 2] = y.z; w[kv][x][nb - 1] = y.w;
            } else {
              const uint2 y = *reinterpret_cast<const uint2*>(src);
              w[kv][x][0] = y.x; w[kv][x][1] = y.y;
            }
          }
        float u[2][nb];  // 2^(127 + kUp - ref)
#pragma unroll
        for (int b = 0; b < nb; ++b) {
          u[0][b] = __uint_as_float((127 + 127 + kUp - ref.x) << 23);
          u[1][b] = __uint_as_float((127 + 127 + kUp - half_of(b % 2 ? ref.w : ref.z, b / 2)) << 23);
        }
        ok = step < kSlots || wait_slot(bar.kv_empty, step - kSlots, 1);
        if (!ok) break;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const uint32_t dst = (kv ? M::kOffV : M::kOffK) + st * M::kOperand + at;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (kv && (ref.y & 1u)) cw[kv][x] &= ~__vcmpeq4(cw[kv][x], 0xFFFFFFFFu);
            float f[nb];
            codes<nb>(cw[kv][x], f);
#pragma unroll
            for (int b = 0; b < nb; ++b) {
              const uint32_t h = pack_half(f[b] * u[kv][b], f[b] * u[kv][b]);
              // values: pieces 2t and 2t + 1 of a block make its 8 elements
              const uint32_t e = kv ? __byte_perm(w[kv][x][b / 2], w[kv][x][nb / 2 + b / 2], b % 2 ? 0x7632 : 0x5410)
                                    : w[kv][x][b];
              uint32_t o[4];
              e2m1x8(e, o);
              // chunk 4b + t of the row
              *reinterpret_cast<uint4*>(smem + (b % 2 ? dst ^ 64u : dst) + (b / 2) * (kTok * 128) + x * 1024) =
                  make_uint4(mul_half2(o[0], h), mul_half2(o[1], h), mul_half2(o[2], h), mul_half2(o[3], h));
            }
          }
        }
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tc::mbar_arrive(&bar.kv_full[st]);
          tc::mbar_arrive(&bar.raw_empty[st]);
        }
      }
      if (lane == 0) tc::mbar_arrive(&bar.item_empty[slot]);
      if (!ok || !valid) break;
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    // ---- softmax of tile i: thread = vector
    const int i = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + i * 128, to = tmem + lanes + 256 + i * 128;
    // load the item's query row, scaled to a maximum near 2^15; its scores lack qs 2^-13
    // (a power that keeps qs off the ends of fp32)
    auto load_q = [&](const Item& it) {
      const int v = it.v0 + i * kRows + r;
      uint4 x[D / 8];
      float am = 0.0f;
#pragma unroll
      for (int c = 0; c < D / 8; ++c) x[c] = make_uint4(0u, 0u, 0u, 0u);
      if (v < it.rows * G) {
        const int row = v / G, h = v - row * G;
        const E* q = static_cast<const E*>(a.q) + (it.row0 + row) * a.q_row + (it.g * G + h) * a.q_head;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) x[c] = q8(q + 8 * c, a.q_vec);
      }
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        const uint32_t w[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 f = two_floats<E>(w[k]);
          am = fmaxf(am, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      }
      const int e = max(int(__float_as_uint(am) >> 23) - 127, -100);
      // the rows take the scale's sign; with a scale of zero all scores are zero
      float f = __uint_as_float(uint32_t(127 + 14 - e) << 23);
      f = a.scale == 0.0f ? 0.0f : copysignf(f, a.scale);
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        const uint32_t w[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
        uint32_t h[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 y = two_floats<E>(w[k]);
          h[k] = pack_half(y.x * f, y.y * f);
        }
        *reinterpret_cast<uint4*>(smem + i * M::kQ + operand_at<kRows>(r, c)) =
            make_uint4(h[0], h[1], h[2], h[3]);
      }
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&bar.q_full[i]);
      return fabsf(a.scale) * 1.44269504088896341f * __uint_as_float(uint32_t(127 - 14 + 13 + e) << 23);
    };
    uint32_t step = 0;
    Item it{};
    float qs = 0.0f;
    bool ok = wait(&bar.item_full[0], 0, 3);
    if (ok) {
      it = s_item[0];
      if (it.valid) qs = load_q(it);
    }
    for (uint32_t n = 0; ok && it.valid; ++n) {
      const int v = it.v0 + i * kRows + r, nv = it.rows * G;
      // tokens, from the part's first on, that this vector sees, that all of the tile see
      const int pos = it.step0 * kTok;
      const int lim = v < nv ? it.len - it.rows + v / G + 1 - pos : 0;
      const int all = it.len - it.rows + (it.v0 + i * kRows) / G + 1 - pos;
      float m = -INFINITY, l = 0.0f, most = 0.0f, far = 0.0f;
      for (int j = 0; j < it.steps; ++j, ++step) {
        const uint32_t buf = step & 1u, tb = ts + buf * 64;
        ok = wait(&bar.s_full[i][buf], step >> 1, 3);
        if (!ok) break;
        tc::tc_fence_after();
        const uint32_t kref = s_ref[step % (4 * kSlots)].x;
        const bool vup = (s_ref[step % (4 * kSlots)].y & 2u) != 0u;
        // not zero: a masked score of -inf has to stay -inf (S is below 2^38: what the
        // bound adds to a score is below 2^-84)
        const float sc = fmaxf(qs * __uint_as_float((127 + kref - 127 - kUp - 13) << 23), 1e-37f);
        most = fmaxf(most, sc);
        uint32_t s[kTok];
#pragma unroll
        for (int c = 0; c < kTok / 32; ++c)
          tc::tmem_ld_32x32b_x32(tb + 32 * c, reinterpret_cast<uint32_t(&)[32]>(s[32 * c]));
        tc::tmem_ld_wait();
        if ((j + 1) * kTok > all) {
          const int keep = lim - j * kTok;
#pragma unroll
          for (int c = 0; c < kTok; ++c)
            if (c >= keep) s[c] = 0xFF800000u;
        }
        float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
        for (int c = 0; c < kTok; c += 4) {
          t0 = fmaxf(fmaxf(t0, __uint_as_float(s[c])), __uint_as_float(s[c + 1]));
          t1 = fmaxf(fmaxf(t1, __uint_as_float(s[c + 2])), __uint_as_float(s[c + 3]));
        }
        const float top = fmaxf(t0, t1) * sc;
        const bool up = top > m + kLazy;
        if (__any_sync(0xffffffffu, up) || vup) {
          const float c = up ? ex2(m - top) : 1.0f;
          if (up) m = top;
          l *= c;
          if (j > 0) {
            // the products of the step before (those before that are complete: these
            // scores came after them)
            ok = wait(&bar.o_done[i][buf ^ 1u], (step - 1) >> 1, 3);
            if (!ok) break;
            tc::tc_fence_after();
#pragma unroll 1
            for (int x = 0; x < D / 16; ++x) {
              float cv = c;
              if (vup) {
                const int b = x / 2;
                const uint4 now = s_ref[step % (4 * kSlots)], then = s_ref[(step - 1) % (4 * kSlots)];
                const uint32_t moved = half_of(b % 2 ? now.w - then.w : now.z - then.z, b / 2);
                cv *= __uint_as_float(uint32_t(max(127 - int(moved), 0)) << 23);
              }
              uint32_t o[16];
              tc::tmem_ld_32x32b_x16(to + 16 * x, o);
              tc::tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * cv);
              tmem_st_x16(to + 16 * x, o);
            }
          }
        }
        const float b0 = kShift - (m == -INFINITY ? 0.0f : m);
        far = fmaxf(far, fabsf(b0));
        const float2 sc2 = make_float2(sc, sc), b2 = make_float2(b0, b0);
        float2 sum0 = make_float2(0.f, 0.f), sum1 = make_float2(0.f, 0.f);
#pragma unroll
        for (int h = 0; h < kTok / 32; ++h) {
          uint32_t p[16];
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            float2 x = make_float2(__uint_as_float(s[32 * h + 2 * c]), __uint_as_float(s[32 * h + 2 * c + 1]));
            x = fma2(x, sc2, b2);
            x.x = ex2(x.x);
            x.y = ex2(x.y);
            if (c & 1) sum1 = add2(sum1, x);
            else sum0 = add2(sum0, x);
            p[c] = pack_half(x.x, x.y);
          }
          tmem_st_x16(tb + 16 * h, p);
        }
        sum0 = add2(sum0, sum1);
        l += sum0.x + sum0.y;
        tmem_st_wait();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&bar.p_full[i][buf]);
      }
      if (!ok) break;
      // the next item's rows before this one's sums: its scores can begin
      Item nx{};
      float nqs = 0.0f;
      ok = wait(&bar.item_full[(n + 1) & 1u], (n + 1) >> 1, 3);
      if (!ok) break;
      nx = s_item[(n + 1) & 1u];
      if (nx.valid) nqs = load_q(nx);
      ok = wait(&bar.o_done[i][(step - 1) & 1u], (step - 1) >> 1, 3);
      if (!ok) break;
      tc::tc_fence_after();
      const uint4 ref = s_ref[(step - 1) % (4 * kSlots)];
      const float nan = __uint_as_float(0x7FC00000u);
      E* out = static_cast<E*>(a.out) +
               ((long long)(it.row0 + v / G) * a.Hq + it.g * G + v % G) * D;
      // Vectors that some values are lost to, whose scores are huge, or whose keys of a
      // step are so strong that what others lose in fp16 would count (rare: S, of which
      // an operand below its range takes 2^-3 at most, is scaled by sc): once more, by
      // the warp.
      bool redo = v < nv && (s_far[n & 1u] != 0 || out_of_range(far) || most > 0x1p-12f);
      auto again = [&] {
        unsigned left = __ballot_sync(0xffffffffu, redo);
        if (left == 0) return;
        if (lane == 0) tc::cta_busy(1);
        for (; left; left &= left - 1) {
          const int x = __shfl_sync(0xffffffffu, v, __ffs(left) - 1);
          attend_exactly<E, D>(a, it.seq, it.row0 + x / G, it.g * G + x % G, it.len - it.rows + x / G + 1);
        }
        if (lane == 0) tc::cta_busy(-1);
      };
      // a part leaves [D + 2][256 vectors]: its own outputs (a sum of values near the end
      // of fp32 has no room for the weights), their maximum and sum of weights
      float* sums = a.part + size_t(it.index) * (256 * (D + 2)) + i * kRows + r;
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
      for (int x = 0; x < D / 32; ++x) {
        uint32_t o[32];
        tc::tmem_ld_32x32b_x32(to + 32 * x, o);
        tc::tmem_ld_wait();
        const bool bad = lim + pos > s_nan[n & 1u][x];
        const float unit = __uint_as_float((half_of(x % 2 ? ref.w : ref.z, x / 2) - kUp) << 23);  // O's: 2^(ref - 127 - kUp)
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(bad ? nan : __uint_as_float(o[k]) * inv * unit);
        if (it.parts > 1) {
#pragma unroll
          for (int k = 0; k < 32; ++k) __stcg(sums + (32 * x + k) * 256, __uint_as_float(o[k]));
        } else if (v < nv && !redo) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            __align__(16) E y[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] = E(__uint_as_float(o[8 * c + k]));
            *reinterpret_cast<uint4*>(out + 32 * x + 8 * c) = *reinterpret_cast<const uint4*>(y);
          }
        }
      }
      if (it.parts == 1) {
        again();
      } else {
        __stcg(sums + D * 256, redo ? INFINITY : m);
        __stcg(sums + (D + 1) * 256, l);
        __threadfence();
        __syncwarp();
        unsigned last = 0;
        if (lane == 0) {
          unsigned* c = a.counters + kPartCounters + (it.index - it.part) * 8 + warp;
          last = atomicInc(c, it.parts - 1) == unsigned(it.parts - 1);
          __threadfence();
        }
        last = __shfl_sync(0xffffffffu, last, 0);
        if (last) {  // the last of the parts' warps with these vectors joins them, in the parts' order
          const float* from = sums - size_t(it.part) * (256 * (D + 2));
          auto at = [&](int part, int c) { return __ldcg(from + size_t(part) * (256 * (D + 2)) + c * 256); };
          float top = -INFINITY, sum = 0.0f, w[kMaxParts];
#pragma unroll
          for (int k = 0; k < kMaxParts; ++k) {
            w[k] = k < it.parts ? at(k, D) : -INFINITY;
            top = fmaxf(top, w[k]);
          }
#pragma unroll
          for (int k = 0; k < kMaxParts; ++k) {
            w[k] = k < it.parts ? ex2(w[k] - (top == -INFINITY ? 0.0f : top)) * at(k, D + 1) : 0.0f;
            sum += w[k];
          }
          const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
          for (int k = 0; k < kMaxParts; ++k) w[k] *= scale;
          redo = v < nv && out_of_range(top);
#pragma unroll 1
          for (int c = 0; c < D; c += 8) {
            float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < kMaxParts; ++k)
              if (k < it.parts) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = fmaf(w[k], at(k, c + e), x[e]);
              }
            if (v < nv && !redo) {
              __align__(16) E y[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) y[e] = E(x[e]);
              *reinterpret_cast<uint4*>(out + c) = *reinterpret_cast<const uint4*>(y);
            }
          }
          again();
        }
      }
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&bar.item_empty[n & 1u]);
      it = nx;
      qs = nqs;
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if (warp == 12) tc::tmem_dealloc(tmem, 512);
}

template <class E, int D>
cudaError_t launch(const AttnArgs& a, cudaStream_t s) {
  const void* fn = reinterpret_cast<const void*>(kv4_attn_many_kernel<E, D>);
  cudaError_t e = ensure_dynamic_smem(fn, Many<D>::kSmem);
  if (e != cudaSuccess) return e;
  // the roles' registers come out of the launch's: never ask for more than it has
  static std::atomic<int> regs{0};
  int have = regs.load(std::memory_order_relaxed);
  if (have == 0) {
    cudaFuncAttributes at;
    e = cudaFuncGetAttributes(&at, fn);
    if (e != cudaSuccess) return e;
    have = (at.numRegs + 7) / 8 * 8;
    regs.store(have, std::memory_order_relaxed);
  }
  if (4 * have < 2 * kRegsSoftmax + kRegsDecode + kRegsOther) return cudaErrorLaunchOutOfResources;
  kv4_attn_many_kernel<E, D><<<kCtas, kThreads, Many<D>::kSmem, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv4_prefill(const kv4::AttnArgs& a, bool bf16, int D, cudaStream_t s) {
  if (bf16)
    return D == 128 ? launch<__nv_bfloat16, 128>(a, s) : launch<__nv_bfloat16, 64>(a, s);
  return D == 128 ? launch<__half, 128>(a, s) : launch<__half, 64>(a, s);
}

}  // namespace mfi
