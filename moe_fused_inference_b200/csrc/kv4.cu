// kv4.cu — the paged 4-bit KV cache: quantising write and read-back.
//
// No reference counterpart: the reference's cache is FP8, one contiguous
// buffer of one sequence (src/ext/mxfp4_decode.cu:440-490).  Layout and codes:
// kv4.cuh.
#include <cuda_fp16.h>

#include "../../include/moe_fp4.h"
#include "kv4.cuh"
#include "work.cuh"

namespace mfi {
namespace {

// Where a call's tokens are.
struct Slots {
  const long long* slots;       // (T,); negative: none
  int* err;
  int capacity;                 // tokens of the pool
  int T, Hkv, page;
  int page_shift;               // log2 of the page, -1 if that is no power of two
};

struct WriteArgs {
  const void* x[2];             // keys, values
  long long row[2], head[2];    // strides in elements (the innermost is 1)
  uint8_t* pool;
  Slots s;
};

struct ReadArgs {
  const uint8_t* pool;
  void* y[2];                   // keys, values (T, Hkv, D)
  Slots s;
};

// A slot as a token of the pool, 0 for one that is none (`live` says which).  No
// branch hangs on the slot before a thread's other loads are on their way.
__device__ __forceinline__ int token_of(const Slots& s, long long slot, bool& live) {
  live = slot >= 0 && slot < s.capacity;
  return live ? int(slot) : 0;
}

// Byte offset in the pool of the tile of (slot, head h of Hkv); row: its row there.
template <int D>
__device__ __forceinline__ long long tile_of(const Slots& s, int slot, int h, int Hkv, int& row) {
  const int pg = s.page_shift >= 0 ? slot >> s.page_shift : slot / s.page;
  const int in = slot - pg * s.page;
  row = in % kv4::kTile;
  return ((long long)pg * Hkv + h) * kv4::head_bytes(D, s.page) +
         (long long)(in / kv4::kTile) * kv4::tile_bytes(D);
}

template <class E>
__device__ __forceinline__ float to_float(E x);
template <>
__device__ __forceinline__ float to_float(float x) { return x; }
template <>
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class E>
__device__ __forceinline__ E from_float(float x);
template <>
__device__ __forceinline__ float from_float(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }

// 8 consecutive elements; kVec: p is 16-byte aligned.
template <class E, bool kVec>
__device__ __forceinline__ void load8(const E* p, float (&v)[8]) {
  if (kVec) {
    constexpr int kPer = 16 / sizeof(E);
#pragma unroll
    for (int i = 0; i < 8 / kPer; ++i) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(p) + i);
      const E* e = reinterpret_cast<const E*>(&raw);
#pragma unroll
      for (int j = 0; j < kPer; ++j) v[i * kPer + j] = to_float(e[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_float(p[j]);
  }
}

// The quad of lanes that holds a block (lane t: elements 8t .. 8t+7): the
// lane's 8 nibbles, and the block's code.
__device__ __forceinline__ uint32_t quantise8(const float (&v)[8], uint8_t& code) {
  float am = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) am = fmax_nan(am, fabsf(v[j]));
  am = fmax_nan(am, __shfl_xor_sync(0xffffffffu, am, 1));
  am = fmax_nan(am, __shfl_xor_sync(0xffffffffu, am, 2));
  const bool finite = am <= 3.402823466e38f;
  const int e = block_exp(am);
  const float inv = __uint_as_float(uint32_t(127 - (finite ? e : 0)) << 23);
  code = finite ? uint8_t(e + 127) : uint8_t(255);
  uint32_t word = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j)  // the sign of v, not of the scaled value: that may underflow
    word |= (e2m1_mag(__fmul_rn(v[j], inv)) | (v[j] < 0.0f ? 8u : 0u)) << (4 * j);
  return finite ? word : 0u;
}

// A block takes kRwThreads / (D/8) tokens of one KV head, its neighbours the other
// heads of the same tokens, so that the rows (T, Hkv, D) are met in order: D/8
// lanes a token, a quad a block of 32 elements, each lane 8 elements of the key
// and of the value.  The tokens of a tile are neighbours in memory: a warp writes
// whole 32-byte sectors.  2 bytes are read (bf16) and 0.53 written an element, but
// what bounds it is instruction issue: some 500 warp instructions for the 16 elements
// of a lane, 80% of the issue slots taken.  16384 tokens of 4 heads of 128, slices of
// a fused projection: 19.9 us, 2.1 TB/s; more tokens a thread do not help (written
// and read back with 1, 2, 4: 28, 27.7, 31.6 us) and cost small calls (1021 tokens of
// 2 heads of 64, fp32, with 1, 2: 3.9, 4.8 us).
constexpr int kRwThreads = 128;

template <class E, int D, bool kVec>
__global__ void __launch_bounds__(kRwThreads) kv4_write_kernel(WriteArgs a) {
  constexpr int kLanes = D / 8, nb = D / 32;
  const int Hkv = a.s.Hkv, run = blockIdx.x / Hkv, h = blockIdx.x - run * Hkv;
  const int t = run * (kRwThreads / kLanes) + threadIdx.x / kLanes, w = threadIdx.x % kLanes;
  const int b = w >> 2, q = w & 3, tt = min(t, a.s.T - 1);
  float k[8], v[8];
  const long long slot = __ldg(a.s.slots + tt);
  load8<E, kVec>(static_cast<const E*>(a.x[0]) + tt * a.row[0] + h * a.head[0] + 8 * w, k);
  load8<E, kVec>(static_cast<const E*>(a.x[1]) + tt * a.row[1] + h * a.head[1] + 8 * w, v);
  uint8_t kc, vc;
  const uint32_t kw = quantise8(k, kc), vw = quantise8(v, vc);
  // value pieces 2q, 2q+1 of blocks b and b ^ 1 make two words of the row: the
  // lane of the even block writes the one of pieces 2q, the odd block's 2q+1
  const uint32_t other = __shfl_xor_sync(0xffffffffu, vw, 4);
  bool live;
  const int token = token_of(a.s, slot, live);
  if (t >= a.s.T) return;
  if (!live) {
    if (slot >= 0) kv4::report(a.s.err, kv4::kErrSlot);
    return;
  }
  int r;
  uint8_t* tile = a.pool + tile_of<D>(a.s, token, h, Hkv, r);
  *reinterpret_cast<uint32_t*>(tile + r * (D / 2) + (q * nb + b) * 4) = kw;
  const uint32_t word = (b & 1) ? __byte_perm(other, vw, 0x7632) : __byte_perm(vw, other, 0x5410);
  const int piece = 2 * q + (b & 1);
  *reinterpret_cast<uint32_t*>(tile + 8 * D + r * (D / 2) + (piece * nb + (b & ~1)) * 2) = word;
  if (q == 0) {
    tile[16 * D + r * nb + b] = kc;
    tile[16 * D + D / 2 + r * nb + b] = vc;
  }
}

// 8 nibbles times a block's scale, rounded once.
template <class E>
__device__ __forceinline__ void store8(E* p, uint32_t w, float s) {
  uint32_t h[4];
  kv4::e2m1x8(w, h);
  __align__(16) E out[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
    out[2 * j] = from_float<E>(f.x * s);
    out[2 * j + 1] = from_float<E>(f.y * s);
  }
#pragma unroll
  for (int j = 0; j < int(sizeof(out) / 16); ++j)
    reinterpret_cast<uint4*>(p)[j] = reinterpret_cast<const uint4*>(out)[j];
}

// The write's shape, the other way round: 0.53 bytes read and 2 written (bf16) an
// element.  The slots, then the rows that they name, are two dependent trips to
// memory.  131072 tokens of 4 heads of 128: 69.6 us, 4.9 TB/s, four bytes written for
// one read; 16384 tokens 9.3 us, 4.6 TB/s.
template <class E, int D>
__global__ void __launch_bounds__(kRwThreads) kv4_read_kernel(ReadArgs a) {
  constexpr int kLanes = D / 8, nb = D / 32;
  const int Hkv = a.s.Hkv, run = blockIdx.x / Hkv, h = blockIdx.x - run * Hkv;
  const int t = run * (kRwThreads / kLanes) + threadIdx.x / kLanes, w = threadIdx.x % kLanes;
  const int b = w >> 2, q = w & 3;
  if (t >= a.s.T) return;
  const long long slot = __ldg(a.s.slots + t);
  bool live;
  int r;
  const int token = token_of(a.s, slot, live);
  const uint8_t* tile = a.pool + tile_of<D>(a.s, token, h, Hkv, r);
  const uint8_t* vr = tile + 8 * D + r * (D / 2);
  uint32_t kw = __ldg(reinterpret_cast<const uint32_t*>(tile + r * (D / 2) + (q * nb + b) * 4));
  uint32_t vw = uint32_t(__ldg(reinterpret_cast<const uint16_t*>(vr + (2 * q * nb + b) * 2))) |
                uint32_t(__ldg(reinterpret_cast<const uint16_t*>(vr + ((2 * q + 1) * nb + b) * 2))) << 16;
  uint32_t kc = __ldg(tile + 16 * D + r * nb + b), vc = __ldg(tile + 16 * D + D / 2 + r * nb + b);
  if (!live) {
    kw = vw = 0u;
    kc = vc = 127u;
    if (slot >= 0) kv4::report(a.s.err, kv4::kErrSlot);
  }
  const long long at = ((long long)t * Hkv + h) * D + 8 * w;
  store8(static_cast<E*>(a.y[0]) + at, kw, kv4::code_value(kc));
  store8(static_cast<E*>(a.y[1]) + at, vw, kv4::code_value(vc));
}

int check_pool(const void* pool, int Hkv, int D, int page, int num_pages) {
  if (D != 64 && D != 128) return set_last_error(MFI_ERR_ARG, "kv4: head_dim must be 64 or 128");
  if (Hkv <= 0 || Hkv > 65535) return set_last_error(MFI_ERR_ARG, "kv4: Hkv must be in [1, 65535]");
  if (page <= 0 || page % kv4::kTile != 0)
    return set_last_error(MFI_ERR_ARG, "kv4: the page must be a positive multiple of 16 tokens");
  if (num_pages <= 0) return set_last_error(MFI_ERR_ARG, "kv4: the pool has no pages");
  if ((long long)num_pages * page > 0x7FFFFFFFLL)
    return set_last_error(MFI_ERR_ARG, "kv4: the pool has more than 2^31 - 1 tokens");
  if (!pool) return set_last_error(MFI_ERR_ARG, "null pointer");
  if (reinterpret_cast<uintptr_t>(pool) & 15)
    return set_last_error(MFI_ERR_ARG, "kv4: the pool must be 16-byte aligned");
  return MFI_OK;
}

int launched() {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MFI_OK : set_last_error(MFI_ERR_CUDA, cudaGetErrorString(e));
}

template <class E>
void launch_write(const WriteArgs& a, int D, bool vec, unsigned grid, cudaStream_t s) {
  if (D == 128) {
    if (vec) kv4_write_kernel<E, 128, true><<<grid, kRwThreads, 0, s>>>(a);
    else kv4_write_kernel<E, 128, false><<<grid, kRwThreads, 0, s>>>(a);
  } else {
    if (vec) kv4_write_kernel<E, 64, true><<<grid, kRwThreads, 0, s>>>(a);
    else kv4_write_kernel<E, 64, false><<<grid, kRwThreads, 0, s>>>(a);
  }
}

template <class E>
void launch_read(const ReadArgs& a, int D, unsigned grid, cudaStream_t s) {
  if (D == 128) kv4_read_kernel<E, 128><<<grid, kRwThreads, 0, s>>>(a);
  else kv4_read_kernel<E, 64><<<grid, kRwThreads, 0, s>>>(a);
}

Slots make_slots(const int64_t* slots, int T, int Hkv, int page, int num_pages) {
  Slots s{};
  s.slots = reinterpret_cast<const long long*>(slots);
  s.err = device_error_flag();
  s.capacity = num_pages * page;
  s.T = T;
  s.Hkv = Hkv;
  s.page = page;
  s.page_shift = -1;
  for (int i = 4; i < 31; ++i)
    if (page == 1 << i) s.page_shift = i;
  return s;
}

// Blocks of a call; 0: more than a grid holds, or tokens that the last block's count
// of 31 bits would pass.
unsigned rw_grid(int T, int Hkv, int D) {
  const int per = kRwThreads / (D / 8);
  if (T > 0x7FFFFFFF - per) return 0u;
  const long long n = ((long long)T + per - 1) / per * Hkv;
  return n > 0x7FFFFFFFLL ? 0u : unsigned(n);
}

}  // namespace

int kv4_check_pool(const void* pool, int Hkv, int D, int page, int num_pages) {
  return check_pool(pool, Hkv, D, page, num_pages);
}

}  // namespace mfi

extern "C" size_t mfi_kv4_pool_bytes(int num_pages, int page, int Hkv, int D) {
  if ((D != 64 && D != 128) || Hkv <= 0 || page <= 0 || page % mfi::kv4::kTile != 0 || num_pages <= 0)
    return 0;
  return size_t(num_pages) * size_t(Hkv) * size_t(mfi::kv4::head_bytes(D, page));
}

extern "C" int mfi_kv4_write(const void* k, long long k_row, long long k_head, const void* v,
                             long long v_row, long long v_head, int dtype, uint8_t* pool,
                             const int64_t* slots, int T, int Hkv, int D, int page, int num_pages,
                             void* stream) {
  if (T < 0) return mfi::set_last_error(MFI_ERR_ARG, "kv4_write: T must not be negative");
  if (dtype != MFI_F32 && dtype != MFI_F16 && dtype != MFI_BF16)
    return mfi::set_last_error(MFI_ERR_ARG, "kv4_write: dtype must be MFI_F32, MFI_F16 or MFI_BF16");
  const int rc = mfi::check_pool(pool, Hkv, D, page, num_pages);
  if (rc != MFI_OK) return rc;
  if (T == 0) return MFI_OK;
  if (!k || !v || !slots) return mfi::set_last_error(MFI_ERR_ARG, "null pointer");
  const unsigned grid = mfi::rw_grid(T, Hkv, D);
  if (grid == 0) return mfi::set_last_error(MFI_ERR_ARG, "kv4_write: too many rows");
  mfi::WriteArgs a{};
  a.x[0] = k; a.x[1] = v;
  a.row[0] = k_row; a.row[1] = v_row;
  a.head[0] = k_head; a.head[1] = v_head;
  a.pool = pool;
  a.s = mfi::make_slots(slots, T, Hkv, page, num_pages);
  // 16-byte loads where every vector starts on a 16-byte boundary
  const int size = dtype == MFI_F32 ? 4 : 2;
  bool vec = true;
  for (int i = 0; i < 2; ++i)
    vec = vec && !((reinterpret_cast<uintptr_t>(a.x[i]) | uintptr_t(a.row[i] * size) |
                    uintptr_t(a.head[i] * size)) & 15);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == MFI_F32) mfi::launch_write<float>(a, D, vec, grid, s);
  else if (dtype == MFI_F16) mfi::launch_write<__half>(a, D, vec, grid, s);
  else mfi::launch_write<__nv_bfloat16>(a, D, vec, grid, s);
  return mfi::launched();
}

extern "C" int mfi_kv4_read(const uint8_t* pool, const int64_t* slots, void* k, void* v, int dtype,
                            int T, int Hkv, int D, int page, int num_pages, void* stream) {
  if (T < 0) return mfi::set_last_error(MFI_ERR_ARG, "kv4_read: T must not be negative");
  if (dtype != MFI_F32 && dtype != MFI_F16 && dtype != MFI_BF16)
    return mfi::set_last_error(MFI_ERR_ARG, "kv4_read: dtype must be MFI_F32, MFI_F16 or MFI_BF16");
  const int rc = mfi::check_pool(pool, Hkv, D, page, num_pages);
  if (rc != MFI_OK) return rc;
  if (T == 0) return MFI_OK;
  if (!k || !v || !slots) return mfi::set_last_error(MFI_ERR_ARG, "null pointer");
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15)
    return mfi::set_last_error(MFI_ERR_ARG, "kv4_read: k and v must be 16-byte aligned");
  const unsigned grid = mfi::rw_grid(T, Hkv, D);
  if (grid == 0) return mfi::set_last_error(MFI_ERR_ARG, "kv4_read: too many rows");
  mfi::ReadArgs a{};
  a.pool = pool;
  a.y[0] = k; a.y[1] = v;
  a.s = mfi::make_slots(slots, T, Hkv, page, num_pages);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == MFI_F32) mfi::launch_read<float>(a, D, grid, s);
  else if (dtype == MFI_F16) mfi::launch_read<__half>(a, D, grid, s);
  else mfi::launch_read<__nv_bfloat16>(a, D, grid, s);
  return mfi::launched();
}
