// kv4_attn.cu — attention over the paged 4-bit KV cache (layout: kv4.cuh).
//
// Sequence i owns the query rows cu_q[i] .. cu_q[i+1] - 1 (i max_q .. without
// cu_q) and the first kv_lens[i] tokens of the pages table[i]; its rows are
// the last of these tokens: row r of R sees tokens 0 .. L - R + r.
//   o = sum_p e^(s_p - m) v_p / sum_p e^(s_p - m),  s_p = scale q . k_p,  m = max s_p
// and zeros for a row that sees no token.
#include <cuda_fp16.h>

#include "../../include/moe_fp4.h"
#include "kv4.cuh"
#include "work.cuh"

namespace mfi {

int kv4_check_pool(const void* pool, int Hkv, int D, int page, int num_pages);

namespace {

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
  int T, max_q, n_seq, Hq, Hkv, page, num_pages, width;
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
    kv4::report(a.err, kv4::kErrPage);
    s.rows = 0;
  }
  if (s.len > room || s.len < 0) {
    kv4::report(a.err, kv4::kErrPage);
    s.len = s.len < 0 ? 0 : int(room);
  }
  return s;
}

__device__ __forceinline__ const uint8_t* tile_at(const AttnArgs& a, int seq, int head, int pos,
                                                  int D) {
  const int p = pos / a.page, in = pos - p * a.page;
  int id = a.table[seq * a.table_ld + p];
  if (id < 0 || id >= a.num_pages) {
    kv4::report(a.err, kv4::kErrPage);
    id = 0;
  }
  return a.pool + ((long long)id * a.Hkv + head) * kv4::head_bytes(D, a.page) +
         (long long)(in / kv4::kTile) * kv4::tile_bytes(D);
}

// One warp per (sequence, row, query head); lane = token for the scores, lane
// = D/32 elements for the sum.
template <class E, int D>
__global__ void __launch_bounds__(128) kv4_attn_kernel(AttnArgs a) {
  constexpr int nb = D / 32;
  __shared__ float s_q[4][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = blockIdx.x * 4LL + warp;
  const int head = int(item % a.Hq);
  const int r = int(item / a.Hq % a.max_q);
  const int i = int(item / a.Hq / a.max_q);
  if (i >= a.n_seq) return;
  const Seq s = sequence(a, i);
  if (r >= s.rows) return;
  const int kvh = head / (a.Hq / a.Hkv);
  const E* q = static_cast<const E*>(a.q) + (s.row0 + r) * a.q_row + head * a.q_head;
  for (int d = lane; d < D; d += 32) s_q[warp][d] = float(q[d]) * a.scale;
  __syncwarp();
  const int see = s.len - s.rows + r + 1;  // tokens this row sees
  float m = -INFINITY, l = 0.0f, o[nb];
#pragma unroll
  for (int b = 0; b < nb; ++b) o[b] = 0.0f;
  for (int p0 = 0; p0 < see; p0 += 32) {
    const int p = p0 + lane;
    float x = -INFINITY;
    if (p < see) {
      const uint8_t* tile = tile_at(a, i, kvh, p, D);
      const int row = p % kv4::kTile;
      const uint32_t* kw = reinterpret_cast<const uint32_t*>(tile + row * (D / 2));
      x = 0.0f;
      for (int b = 0; b < nb; ++b) {
        float dot = 0.0f;
        for (int t = 0; t < 4; ++t) {
          const uint32_t w = kw[t * nb + b];
#pragma unroll
          for (int j = 0; j < 8; ++j)
            dot = fmaf(kv4::nibble_value(w >> (4 * j)), s_q[warp][32 * b + 8 * t + j], dot);
        }
        x = fmaf(dot, kv4::code_value(tile[16 * D + row * nb + b]), x);
      }
    }
    float mx = x;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) mx = fmax_nan(mx, __shfl_xor_sync(0xffffffffu, mx, off));
    const float nm = fmax_nan(m, mx);
    const float ref = nm == -INFINITY ? 0.0f : nm;
    const float corr = expf(m - ref), pr = expf(x - ref);
    m = nm;
    float sum = pr;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    l = l * corr + sum;
#pragma unroll
    for (int b = 0; b < nb; ++b) o[b] *= corr;
    for (int j = 0; j < 32 && p0 + j < see; ++j) {
      const float pj = __shfl_sync(0xffffffffu, pr, j);
      const uint8_t* tile = tile_at(a, i, kvh, p0 + j, D);
      const int row = (p0 + j) % kv4::kTile;
      const uint8_t* vr = tile + 8 * D + row * (D / 2);
      // lane = element of each block: piece lane / 4, nibble lane % 4
#pragma unroll
      for (int b = 0; b < nb; ++b) {
        const uint8_t byte = vr[((lane >> 2) * nb + b) * 2 + ((lane & 3) >> 1)];
        const float v = kv4::nibble_value(uint32_t(byte) >> (4 * (lane & 1))) *
                        kv4::code_value(tile[16 * D + D / 2 + row * nb + b]);
        o[b] = fmaf(pj, v, o[b]);
      }
    }
  }
  E* out = static_cast<E*>(a.out) + ((long long)(s.row0 + r) * a.Hq + head) * D;
#pragma unroll
  for (int b = 0; b < nb; ++b) out[32 * b + lane] = E(l == 0.0f ? 0.0f : o[b] / l);
}

}  // namespace
}  // namespace mfi

extern "C" size_t mfi_kv4_attn_workspace_bytes(int n_seq, int Hq, int Hkv, int D, int max_q) {
  if (n_seq <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || (D != 64 && D != 128) || max_q <= 0)
    return 0;
  return 256;
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
  if (!q || !table || !kv_lens || !out || !workspace)
    return mfi::set_last_error(MFI_ERR_ARG, "null pointer");
  if (workspace_bytes < mfi_kv4_attn_workspace_bytes(n_seq, Hq, Hkv, D, max_q))
    return mfi::set_last_error(MFI_ERR_WORKSPACE, "workspace smaller than the kv4_attn workspace query");
  mfi::AttnArgs a{};
  a.q = q; a.q_row = q_row; a.q_head = q_head;
  a.pool = pool; a.table = table; a.table_ld = table_ld;
  a.kv_lens = kv_lens; a.cu_q = cu_q; a.out = out;
  a.err = mfi::device_error_flag();
  a.T = T; a.max_q = max_q; a.n_seq = n_seq; a.Hq = Hq; a.Hkv = Hkv;
  a.page = page; a.num_pages = num_pages; a.width = width;
  a.scale = scale;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const long long blocks = ((long long)n_seq * max_q * Hq + 3) / 4;
  if (blocks > 0x7FFFFFFFLL) return mfi::set_last_error(MFI_ERR_ARG, "kv4_attn: too many rows");
  const unsigned g = unsigned(blocks);
  if (dtype == MFI_BF16) {
    if (D == 128) mfi::kv4_attn_kernel<__nv_bfloat16, 128><<<g, 128, 0, s>>>(a);
    else mfi::kv4_attn_kernel<__nv_bfloat16, 64><<<g, 128, 0, s>>>(a);
  } else {
    if (D == 128) mfi::kv4_attn_kernel<__half, 128><<<g, 128, 0, s>>>(a);
    else mfi::kv4_attn_kernel<__half, 64><<<g, 128, 0, s>>>(a);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MFI_OK : mfi::set_last_error(MFI_ERR_CUDA, cudaGetErrorString(e));
}
