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

struct WriteArgs {
  const void* x[2];             // keys, values
  long long row[2], head[2];    // strides in elements (the innermost is 1)
  uint8_t* pool;
  const long long* slots;       // (T,), negative: skip the row
  int* err;
  long long capacity;           // tokens of the pool
  int T, Hkv, page;
};

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

__device__ __forceinline__ uint8_t* tile_of(uint8_t* pool, long long slot, int h, int Hkv, int page,
                                            int D) {
  const long long pg = slot / page;
  const int in = int(slot - pg * page);
  return pool + (pg * Hkv + h) * kv4::head_bytes(D, page) +
         (long long)(in / kv4::kTile) * kv4::tile_bytes(D);
}

// One lane per 8 elements (a quad per block): lanes run over the elements,
// then heads, then key / value, then tokens.
template <class E, int D, bool kVec>
__global__ void __launch_bounds__(256) kv4_write_kernel(WriteArgs a) {
  constexpr int kLanes = D / 8, nb = D / 32;
  const long long i = blockIdx.x * 256LL + threadIdx.x;
  const int w = int(i % kLanes);
  const long long vec = i / kLanes;  // (token, key / value, head)
  const int h = int(vec % a.Hkv);
  const int kv = int(vec / a.Hkv) & 1;
  const long long tok = vec / a.Hkv / 2;
  const bool live = tok < a.T;
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (live)
    load8<E, kVec>(static_cast<const E*>(a.x[kv]) + tok * a.row[kv] + h * a.head[kv] + 8 * w, v);
  float am = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) am = fmax_nan(am, fabsf(v[j]));
  am = fmax_nan(am, __shfl_xor_sync(0xffffffffu, am, 1));
  am = fmax_nan(am, __shfl_xor_sync(0xffffffffu, am, 2));
  const bool finite = am <= 3.402823466e38f;
  const int e = block_exp(am);
  const float inv = __uint_as_float(uint32_t(127 - (finite ? e : 0)) << 23);
  uint32_t word = 0;
  if (finite) {
#pragma unroll
    for (int j = 0; j < 8; ++j)  // the sign of v, not of the scaled value: that may underflow
      word |= (e2m1_mag(__fmul_rn(v[j], inv)) | (v[j] < 0.0f ? 8u : 0u)) << (4 * j);
  }
  if (!live) return;
  const long long slot = a.slots[tok];
  if (slot < 0) return;
  if (slot >= a.capacity) {
    kv4::report(a.err, kv4::kErrSlot);
    return;
  }
  uint8_t* tile = tile_of(a.pool, slot, h, a.Hkv, a.page, D);
  const int r = int(slot % kv4::kTile);
  const int b = w >> 2, t = w & 3;
  uint8_t* rowp = tile + kv * 8 * D + r * (D / 2);
  if (kv == 0) {
    *reinterpret_cast<uint32_t*>(rowp + (t * nb + b) * 4) = word;
  } else {
    *reinterpret_cast<uint16_t*>(rowp + ((2 * t) * nb + b) * 2) = uint16_t(word);
    *reinterpret_cast<uint16_t*>(rowp + ((2 * t + 1) * nb + b) * 2) = uint16_t(word >> 16);
  }
  if (t == 0) tile[16 * D + kv * (D / 2) + r * nb + b] = finite ? uint8_t(e + 127) : uint8_t(255);
}

struct ReadArgs {
  const uint8_t* pool;
  const long long* slots;
  void* y[2];                   // keys, values (T, Hkv, D)
  int* err;
  long long capacity;
  int T, Hkv, page;
};

template <class E, int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(ReadArgs a) {
  constexpr int kLanes = D / 8, nb = D / 32;
  const long long i = blockIdx.x * 256LL + threadIdx.x;
  const int w = int(i % kLanes);
  const long long vec = i / kLanes;
  const int h = int(vec % a.Hkv);
  const int kv = int(vec / a.Hkv) & 1;
  const long long tok = vec / a.Hkv / 2;
  if (tok >= a.T) return;
  const long long slot = a.slots[tok];
  uint32_t word = 0;
  float s = 1.0f;
  if (slot >= a.capacity) kv4::report(a.err, kv4::kErrSlot);
  if (slot >= 0 && slot < a.capacity) {
    const uint8_t* tile =
        tile_of(const_cast<uint8_t*>(a.pool), slot, h, a.Hkv, a.page, D);
    const int r = int(slot % kv4::kTile);
    const int b = w >> 2, t = w & 3;
    const uint8_t* rowp = tile + kv * 8 * D + r * (D / 2);
    if (kv == 0)
      word = *reinterpret_cast<const uint32_t*>(rowp + (t * nb + b) * 4);
    else
      word = uint32_t(*reinterpret_cast<const uint16_t*>(rowp + ((2 * t) * nb + b) * 2)) |
             uint32_t(*reinterpret_cast<const uint16_t*>(rowp + ((2 * t + 1) * nb + b) * 2)) << 16;
    s = kv4::code_value(tile[16 * D + kv * (D / 2) + r * nb + b]);
  }
  __align__(16) E out[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) out[j] = from_float<E>(kv4::nibble_value(word >> (4 * j)) * s);
  E* y = static_cast<E*>(a.y[kv]) + (tok * a.Hkv + h) * D + 8 * w;
#pragma unroll
  for (int j = 0; j < int(sizeof(out) / 16); ++j)
    reinterpret_cast<uint4*>(y)[j] = reinterpret_cast<const uint4*>(out)[j];
}

int check_pool(const void* pool, int Hkv, int D, int page, int num_pages) {
  if (D != 64 && D != 128) return set_last_error(MFI_ERR_ARG, "kv4: head_dim must be 64 or 128");
  if (Hkv <= 0 || Hkv > 65535) return set_last_error(MFI_ERR_ARG, "kv4: Hkv must be in [1, 65535]");
  if (page <= 0 || page % kv4::kTile != 0)
    return set_last_error(MFI_ERR_ARG, "kv4: the page must be a positive multiple of 16 tokens");
  if (num_pages <= 0) return set_last_error(MFI_ERR_ARG, "kv4: the pool has no pages");
  if (!pool) return set_last_error(MFI_ERR_ARG, "null pointer");
  if (reinterpret_cast<uintptr_t>(pool) & 15)
    return set_last_error(MFI_ERR_ARG, "kv4: the pool must be 16-byte aligned");
  return MFI_OK;
}

int launched(const char*) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MFI_OK : set_last_error(MFI_ERR_CUDA, cudaGetErrorString(e));
}

template <class E>
void launch_write(const WriteArgs& a, int D, bool vec, unsigned blocks, cudaStream_t s) {
  if (D == 128) {
    if (vec) kv4_write_kernel<E, 128, true><<<blocks, 256, 0, s>>>(a);
    else kv4_write_kernel<E, 128, false><<<blocks, 256, 0, s>>>(a);
  } else {
    if (vec) kv4_write_kernel<E, 64, true><<<blocks, 256, 0, s>>>(a);
    else kv4_write_kernel<E, 64, false><<<blocks, 256, 0, s>>>(a);
  }
}

template <class E>
void launch_read(const ReadArgs& a, int D, unsigned blocks, cudaStream_t s) {
  if (D == 128) kv4_read_kernel<E, 128><<<blocks, 256, 0, s>>>(a);
  else kv4_read_kernel<E, 64><<<blocks, 256, 0, s>>>(a);
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
  mfi::WriteArgs a{};
  a.x[0] = k; a.x[1] = v;
  a.row[0] = k_row; a.row[1] = v_row;
  a.head[0] = k_head; a.head[1] = v_head;
  a.pool = pool;
  a.slots = reinterpret_cast<const long long*>(slots);
  a.err = mfi::device_error_flag();
  a.capacity = (long long)num_pages * page;
  a.T = T; a.Hkv = Hkv; a.page = page;
  // 16-byte loads where every vector starts on a 16-byte boundary
  const int size = dtype == MFI_F32 ? 4 : 2;
  bool vec = true;
  for (int i = 0; i < 2; ++i)
    vec = vec && !((reinterpret_cast<uintptr_t>(a.x[i]) | uintptr_t(a.row[i] * size) |
                    uintptr_t(a.head[i] * size)) & 15);
  const long long lanes = (long long)T * 2 * Hkv * (D / 8);
  const long long blocks = (lanes + 255) / 256;
  if (blocks > 0x7FFFFFFFLL) return mfi::set_last_error(MFI_ERR_ARG, "kv4_write: too many rows");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == MFI_F32) mfi::launch_write<float>(a, D, vec, unsigned(blocks), s);
  else if (dtype == MFI_F16) mfi::launch_write<__half>(a, D, vec, unsigned(blocks), s);
  else mfi::launch_write<__nv_bfloat16>(a, D, vec, unsigned(blocks), s);
  return mfi::launched("kv4_write");
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
  mfi::ReadArgs a{};
  a.pool = pool;
  a.slots = reinterpret_cast<const long long*>(slots);
  a.y[0] = k; a.y[1] = v;
  a.err = mfi::device_error_flag();
  a.capacity = (long long)num_pages * page;
  a.T = T; a.Hkv = Hkv; a.page = page;
  const long long lanes = (long long)T * 2 * Hkv * (D / 8);
  const long long blocks = (lanes + 255) / 256;
  if (blocks > 0x7FFFFFFFLL) return mfi::set_last_error(MFI_ERR_ARG, "kv4_read: too many rows");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == MFI_F32) mfi::launch_read<float>(a, D, unsigned(blocks), s);
  else if (dtype == MFI_F16) mfi::launch_read<__half>(a, D, unsigned(blocks), s);
  else mfi::launch_read<__nv_bfloat16>(a, D, unsigned(blocks), s);
  return mfi::launched("kv4_read");
}
