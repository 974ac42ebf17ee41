// cq_sparse.cuh -- what the block-sparse attention kernels share: the visible
// blocks of a query, and the device-side length check.
#pragma once

#include "cq_common.cuh"

namespace cq {
namespace sparse {

constexpr int ERR_LENGTH = 4;  // a device-resident length outside [q_len, mapped tokens]
constexpr int kMaxTop = 4096;  // longest block list

// Records a bad device-resident length for cq_device_error (the word of cq_sparse.cu's kernels; cq_sparse_fast.cu has
// its own).
__device__ void set_length_error();

// Cached tokens of a launch: T, or the device-resident length (which must lie
// in [lo, T]: T is then what grid and workspace are sized for).  0: nothing to do.
__device__ __forceinline__ int64_t launch_length(int64_t T, const int64_t *len_dev, int64_t lo) {
  if (!len_dev) return T;
  const int64_t n = *len_dev;
  return (n < lo || n > T) ? 0 : n;
}

// First token a query of sequence b may see (left padding), never negative.
__device__ __forceinline__ int64_t first_token(const int64_t *starts, int b) {
  const int64_t s = starts ? starts[b] : 0;
  return s > 0 ? s : 0;
}

// amax below this counts as a zero query head (its reciprocal would overflow).
constexpr float kTinyQuery = 1e-30f;
// Query values enter the block scores as finite numbers of the fp16 range: NaN counts as 0.
__device__ __forceinline__ float finite_query(float x) { return isnan(x) ? 0.f : fminf(fmaxf(x, -65504.f), 65504.f); }

// Monotone map of a finite or infinite float to an unsigned key.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

}  // namespace sparse

// Attention over listed blocks on the chunk-block layout (cq_sparse_fast.cu);
// it needs no workspace.
bool sparse_fast_supported(const cq_paged_cache &c, int64_t T, int n_q_heads, int block_tokens);
int run_sparse_fast(const cq_paged_cache &c, int64_t T, const int64_t *len_dev, const void *q, int q_dtype,
                    int n_q_heads, int q_len, int64_t q_sb, int64_t q_sh, int64_t q_sq, float scale,
                    const int64_t *starts, const int32_t *blocks, int top, int block_tokens, void *out, int out_dtype,
                    float *lse_out, cudaStream_t st);
int read_sparse_fast_error(int clear);

}  // namespace cq
