// cq_sparse.cu -- sparse attention over the compressed cache: each query token
// attends only to blocks of tokens that a cheap score picks for it.
//
//   cq_block_bounds   per block and channel, the range of the decoded keys as
//                     int8 codes with one fp32 scale per block (2D + 4 bytes
//                     per block and kv-head);
//   cq_block_select   int8 query x int8 range: an upper estimate of the largest
//                     q.k in each block, and the best blocks per query token;
//   cq_sparse_attention  softmax attention over the listed blocks' tokens.
//
// The score of block j for query token i and kv-head h is
//   max over the group's heads g of  (s_g * s_j) * dot_gj,
//   dot_gj = sum_d max(q8_gd * lo_jd, q8_gd * hi_jd)
// with q8 = rint(q * (127 / amax)), s_g = amax / 127.  dot is a sum of whole
// numbers below 2^23 (|q8|, |code| <= 127, D <= 256), so it does not depend on
// the order of summation, and the three roundings after it are fixed: the
// chosen lists are the same for every split of the work.
#include <algorithm>

#include "cq_prefill.cuh"
#include "cq_sparse.cuh"

namespace cq {
namespace sparse {

__device__ int g_sparse_error;
__device__ void set_length_error() { atomicExch(&g_sparse_error, ERR_LENGTH); }

// ---------------------------------------------------------------------------
// bounds: one CTA per (sequence, kv-head, block), a thread per channel
// ---------------------------------------------------------------------------
struct BoundsArgs {
  CacheView cv;
  int64_t t0, T;            // blocks of tokens t0 .. T-1
  const int64_t *len_dev;   // else: of the last S tokens of *len_dev
  int S, bt, nb;            // nb: blocks per unit in the grid
  int8_t *codes;
  float *scales;
  int64_t max_blocks;
};

// The fp16 key of one channel as reconstruct (mode 0) rounds it.
__device__ __forceinline__ float key_f16(const TokLoc &L, int d, int D, int order) {
  const __half a = L.anchor[d];
  if (!L.codes) return __half2float(a);
  const int code = nibble_at(L.codes, d, D, order) - 8;
  return __half2float(__hadd_rn(a, __hmul_rn(__int2half_rn(code), __float2half_rn(L.scale))));
}

// The least whole number c with c * s >= x (s > 0, |x| <= 126 s up to
// rounding): the rounded quotient, corrected by the exact sign of x - c * s.
__device__ __forceinline__ float ceil_code(float x, float s) {
  const float c = rintf(__fdiv_rn(x, s));
  return fmaf(-c, s, x) > 0.f ? c + 1.f : c;
}

// One block's codes and scale from the per-channel range held by `threads`
// threads (channel d of thread d); amax: the block's largest |x|.
__device__ __forceinline__ void store_codes(int8_t *codes, int d, int D, float lo, float hi, float s) {
  float l = 0.f, h = 0.f;
  if (s > 0.f) {
    h = ceil_code(hi, s);
    l = -ceil_code(-lo, s);
  }
  codes[d] = (int8_t)fminf(fmaxf(l, -127.f), 127.f);
  codes[D + d] = (int8_t)fminf(fmaxf(h, -127.f), 127.f);
}

__global__ void __launch_bounds__(256) block_bounds_kernel(BoundsArgs A) {
  __shared__ float s_red[8];
  const CacheView &cv = A.cv;
  int64_t T = A.T, t0 = A.t0;
  if (A.len_dev) {
    T = launch_length(A.T, A.len_dev, A.S);
    if (T == 0) {
      if (blockIdx.x == 0 && threadIdx.x == 0) set_length_error();
      return;
    }
    t0 = T - A.S;
  }
  const int64_t unit = blockIdx.x / A.nb;
  const int64_t j = t0 / A.bt + (int64_t)(blockIdx.x - unit * A.nb);
  if (j * A.bt >= T) return;
  const int b = (int)(unit / cv.H), h = (int)(unit - (int64_t)b * cv.H);
  const int64_t ta = j * A.bt, tb = min(T, ta + A.bt);
  const int d = threadIdx.x;
  float lo = INFINITY, hi = -INFINITY;
  for (int64_t t = ta; t < tb; ++t) {
    const TokLoc L = locate(cv, 0, b, h, t);
    if (d < cv.D) {
      const float x = key_f16(L, d, cv.D, cv.c[0].order);
      lo = fminf(lo, x);  // a NaN is left out
      hi = fmaxf(hi, x);
    }
  }
  // no value at all (every token NaN) counts as 0; infinities as the largest fp16 value
  if (lo > hi) lo = hi = 0.f;
  lo = fminf(fmaxf(lo, -65504.f), 65504.f);
  hi = fminf(fmaxf(hi, -65504.f), 65504.f);
  float amax = warp_max(d < cv.D ? fmaxf(fabsf(lo), fabsf(hi)) : 0.f);
  if ((threadIdx.x & 31) == 0) s_red[threadIdx.x >> 5] = amax;
  __syncthreads();
  amax = 0.f;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) amax = fmaxf(amax, s_red[w]);
  const float s = __fdiv_rn(amax, 126.f);
  const int64_t row = unit * A.max_blocks + j;
  if (d < cv.D) store_codes(A.codes + row * 2 * cv.D, d, cv.D, lo, hi, s);
  if (threadIdx.x == 0) A.scales[row] = s;
}

// out [units][n][2][D] fp32 = code * scale of blocks first .. first + n - 1
__global__ void bounds_read_kernel(const int8_t *codes, const float *scales, int64_t units, int64_t max_blocks,
                                   int64_t first, int64_t n, int D, float *out) {
  const int64_t row = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (row >= units * n) return;
  const int64_t u = row / n, j = first + (row - u * n);
  const int8_t *c = codes + (u * max_blocks + j) * 2 * D;
  const float s = scales[u * max_blocks + j];
  for (int i = threadIdx.x & 31; i < 2 * D; i += 32) out[row * 2 * D + i] = (float)c[i] * s;
}

// ---------------------------------------------------------------------------
// selection
// ---------------------------------------------------------------------------
struct SelectArgs {
  const int8_t *codes;
  const float *scales;
  int64_t max_blocks;
  int bt, B, H, D, G, q_len;
  int64_t T;
  const int64_t *len_dev;
  const void *q;
  int q_dtype;
  int64_t q_sb, q_sh, q_sq;
  const int64_t *starts;
  int first, recent, top;
  int32_t *blocks;
  float *block_scores;
  int64_t n;     // score row length: blocks of T
  float *score;  // [units][q_len][n]
};

// One warp per (unit, query token, block).
__global__ void __launch_bounds__(256) block_score_kernel(SelectArgs A) {
  const int64_t T = launch_length(A.T, A.len_dev, A.q_len);
  if (T == 0) return;
  const int lane = threadIdx.x & 31;
  const int64_t w = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int64_t rows = (int64_t)A.B * A.H * A.q_len;
  const int64_t row = w / A.n, j = w - row * A.n;
  if (row >= rows) return;
  const int i = (int)(row % A.q_len);
  const int64_t unit = row / A.q_len;
  const int b = (int)(unit / A.H), h = (int)(unit - (int64_t)b * A.H);
  if (j > (T - A.q_len + i) / A.bt) return;  // not visible
  const int8_t *c = A.codes + (unit * A.max_blocks + j) * 2 * A.D;
  const float sj = A.scales[unit * A.max_blocks + j];
  float best = -INFINITY;
  for (int g = 0; g < A.G; ++g) {
    const int64_t qb = b * A.q_sb + (int64_t)(h * A.G + g) * A.q_sh + i * A.q_sq;
    float x[8], amax = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int d = lane + 32 * k;
      x[k] = d < A.D ? finite_query(load_as_float(A.q, qb + d, A.q_dtype)) : 0.f;
      amax = fmaxf(amax, fabsf(x[k]));
    }
    amax = warp_max(amax);
    const bool zero = amax < kTinyQuery;
    const float r = zero ? 0.f : __fdiv_rn(127.f, amax);
    int dot = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int d = lane + 32 * k;
      if (d < A.D) {
        const int q8 = (int)rintf(__fmul_rn(x[k], r));
        dot += q8 * (int)(q8 > 0 ? c[A.D + d] : c[d]);
      }
    }
    dot = __reduce_add_sync(0xffffffffu, dot);
    const float sg = zero ? 0.f : __fdiv_rn(amax, 127.f);
    best = fmaxf(best, __fmul_rn(__fmul_rn(sg, sj), (float)dot));
  }
  if (lane == 0) A.score[row * A.n + j] = __fadd_rn(best, 0.f);  // -0 becomes +0: equal scores have equal keys
}

// One CTA per (unit, query token): the `top` best visible blocks.  A radix
// select finds the key of the last one taken (4 passes of 8 bits), and an
// ordered pass writes the list, taking equal keys from the lowest index on.
__global__ void __launch_bounds__(256) block_topk_kernel(SelectArgs A) {
  __shared__ int hist[256];
  __shared__ int s_scan[8], s_scan2[8];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const int64_t T = launch_length(A.T, A.len_dev, A.q_len);
  if (T == 0) {
    if (blockIdx.x == 0 && threadIdx.x == 0) set_length_error();
    return;
  }
  const int64_t row = blockIdx.x;
  const int i = (int)(row % A.q_len);
  const int b = (int)(row / ((int64_t)A.q_len * A.H));
  const int64_t p = T - A.q_len + i;
  const int64_t st = first_token(A.starts, b);
  int32_t *out = A.blocks + row * A.top;
  float *out_s = A.block_scores ? A.block_scores + row * A.top : nullptr;
  const int fb = (int)min(st / A.bt, (int64_t)INT32_MAX), lb = (int)(p / A.bt);
  const int nv = st > p ? 0 : lb - fb + 1;
  const float *score = A.score + row * A.n;
  auto key = [&](int j) -> uint32_t {
    return (j < fb + A.first || j > lb - A.recent) ? 0xffffffffu : order_key(score[j]);
  };
  uint32_t thr = 0;  // keys above it are taken, and s_need of those equal to it
  int need = 0;
  if (nv > A.top) {
    uint32_t prefix = 0;
    need = A.top;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int k = threadIdx.x; k < 256; k += blockDim.x) hist[k] = 0;
      __syncthreads();
      for (int j = fb + threadIdx.x; j <= lb; j += blockDim.x) {
        const uint32_t u = key(j);
        if (shift == 24 || (u >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(u >> shift) & 255], 1);
      }
      __syncthreads();
      if (threadIdx.x == 0) {
        int left = need, k = 255;
        for (; k > 0 && hist[k] < left; --k) left -= hist[k];
        s_prefix = prefix | ((uint32_t)k << shift);
        s_need = left;
      }
      __syncthreads();
      prefix = s_prefix;
      need = s_need;
      __syncthreads();
    }
    thr = prefix;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int done = 0, eq_done = 0;
  for (int base = fb; base < fb + nv; base += blockDim.x) {
    const int j = base + threadIdx.x;
    const bool in = j <= lb;
    const uint32_t u = in ? key(j) : 0u;
    const bool eq = in && nv > A.top && u == thr;
    const unsigned be = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) s_scan2[warp] = __popc(be);
    __syncthreads();
    int eq_before = eq_done + __popc(be & ((1u << lane) - 1u)), eq_all = 0;
    for (int w = 0; w < 8; ++w) {
      if (w < warp) eq_before += s_scan2[w];
      eq_all += s_scan2[w];
    }
    const bool take = in && (nv <= A.top || u > thr || (eq && eq_before < need));
    const unsigned bt = __ballot_sync(0xffffffffu, take);
    if (lane == 0) s_scan[warp] = __popc(bt);
    __syncthreads();
    int at = done + __popc(bt & ((1u << lane) - 1u)), all = 0;
    for (int w = 0; w < 8; ++w) {
      if (w < warp) at += s_scan[w];
      all += s_scan[w];
    }
    if (take) {
      out[at] = j;
      if (out_s) out_s[at] = score[j];
    }
    done += all;
    eq_done += eq_all;
    __syncthreads();
  }
  for (int k = done + threadIdx.x; k < A.top; k += blockDim.x) {
    out[k] = -1;
    if (out_s) out_s[k] = -INFINITY;
  }
}

// ---------------------------------------------------------------------------
// attention over the listed blocks: the general kernel (every layout)
// ---------------------------------------------------------------------------
constexpr int kGenWarps = 4;

struct SparseArgs {
  CacheView cv;
  const void *q;
  int q_dtype, Hq, q_len, top, bt, splits;
  int64_t q_sb, q_sh, q_sq;
  float scale;
  int64_t T;
  const int64_t *len_dev;
  const int64_t *starts;
  const int32_t *blocks;  // [B][H][q_len][top]
  float *ws_m, *ws_l, *ws_o;
};

__device__ __forceinline__ float value_at(const TokLoc &L, int d, int D, int order) {
  const float a = __half2float(L.anchor[d]);
  return L.codes ? fmaf((float)(nibble_at(L.codes, d, D, order) - 8), L.scale, a) : a;
}

// One CTA per (sequence, query head, query token, split of the list); warps
// take tokens in turn, lanes hold dims lane + 32 i.
__global__ void __launch_bounds__(kGenWarps * 32) sparse_generic_kernel(SparseArgs A) {
  __shared__ float s_m[kGenWarps], s_l[kGenWarps];
  __shared__ float s_o[kGenWarps][256];
  const CacheView &cv = A.cv;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sp = (int)(blockIdx.x % A.splits);
  const int64_t row = blockIdx.x / A.splits;
  const int i = (int)(row % A.q_len);
  const int hq = (int)((row / A.q_len) % A.Hq);
  const int b = (int)(row / ((int64_t)A.q_len * A.Hq));
  const int D = cv.D, h = hq / (A.Hq / cv.H);
  const int64_t T = launch_length(A.T, A.len_dev, A.q_len);
  if (T == 0 && blockIdx.x == 0 && threadIdx.x == 0) set_length_error();
  const int64_t p = T - A.q_len + i, st = first_token(A.starts, b);
  const int32_t *list = A.blocks + (((int64_t)b * cv.H + h) * A.q_len + i) * A.top;
  const int per = (A.top + A.splits - 1) / A.splits;
  const int s0 = sp * per, s1 = T == 0 ? s0 : min(A.top, s0 + per);

  float qv[8];
  const float sc = round_dt(A.scale, A.q_dtype);
  const int64_t qb = b * A.q_sb + hq * A.q_sh + i * A.q_sq;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int d = lane + 32 * k;
    qv[k] = d < D ? round_dt(load_as_float(A.q, qb + d, A.q_dtype) * sc, A.q_dtype) : 0.f;
  }
  float m = -INFINITY, l = 0.f, acc[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) acc[k] = 0.f;
  for (int s = s0; s < s1; ++s) {
    const int64_t j = list[s];
    if (j < 0 || (s > 0 && j <= list[s - 1])) continue;  // absent, or a repeat
    const int64_t ta = max(st, j * A.bt), tb = min(p + 1, (j + 1) * A.bt);
    for (int64_t t = ta + warp; t < tb; t += kGenWarps) {
      const TokLoc K = locate(cv, 0, b, h, t);
      float part = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int d = lane + 32 * k;
        if (d < D) part = fmaf(qv[k], value_at(K, d, D, cv.c[0].order), part);
      }
      const float x = warp_sum(part);
      const float mn = fmaxf(m, x);
      const float f = mn == -INFINITY ? 1.f : expf(m - mn);
      const float pr = mn == -INFINITY ? 0.f : expf(x - mn);
      m = mn;
      l = l * f + pr;
      const TokLoc V = locate(cv, 1, b, h, t);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int d = lane + 32 * k;
        if (d < D) acc[k] = fmaf(pr, value_at(V, d, D, cv.c[1].order), acc[k] * f);
      }
    }
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (lane + 32 * k < D) s_o[warp][lane + 32 * k] = acc[k];
  __syncthreads();
  if (warp != 0) return;
  float M = -INFINITY, L = 0.f, fw[kGenWarps];
  for (int w = 0; w < kGenWarps; ++w) M = fmaxf(M, s_m[w]);
  for (int w = 0; w < kGenWarps; ++w) {
    fw[w] = s_m[w] == -INFINITY ? 0.f : expf(s_m[w] - M);
    L += s_l[w] * fw[w];
  }
  const int64_t o = row * A.splits + sp;
  if (lane == 0) {
    A.ws_m[o] = M;
    A.ws_l[o] = L;
  }
  for (int d = lane; d < D; d += 32) {
    float v = 0.f;
    for (int w = 0; w < kGenWarps; ++w) v += s_o[w][d] * fw[w];
    A.ws_o[o * D + d] = v;
  }
}

// Splits of the block list: enough CTAs for the machine, at least one block each.
static int pick_list_splits(int64_t rows, int top) {
  const int64_t want = (2 * 148 * 4 + rows - 1) / rows;
  return (int)std::max<int64_t>(1, std::min<int64_t>(want, std::min(top, 64)));
}

static size_t generic_bytes(int64_t rows, int splits, int D) { return (size_t)rows * splits * (2 + D) * sizeof(float); }

}  // namespace sparse

int read_sparse_error(int clear) {
  int v = 0;
  cudaMemcpyFromSymbol(&v, sparse::g_sparse_error, sizeof(int));
  if (clear && v) {
    const int z = 0;
    cudaMemcpyToSymbol(sparse::g_sparse_error, &z, sizeof(int));
  }
  const int f = read_sparse_fast_error(clear);
  return v ? v : f;
}
int read_bounds_error_sparse(int clear) { return read_bounds_error_here(clear); }

}  // namespace cq

using namespace cq;

static int bounds_checks(const cq_paged_cache *cache, int64_t T, int32_t bt, const void *codes, const void *scales,
                         int64_t max_blocks, const char *what) {
  int r = validate_cache(cache);
  if (r) return r;
  const std::string w(what);
  CQ_REQUIRE(codes && scales, CQ_ERR_INVALID, w + ": null pointer");
  CQ_REQUIRE(bt >= 1, CQ_ERR_INVALID, w + ": block_tokens must be >= 1");
  CQ_REQUIRE(T >= 1 && (T + cache->page_tokens - 1) / cache->page_tokens <= cache->max_pages, CQ_ERR_INVALID,
             w + ": tokens beyond the mapped pages (or none)");
  CQ_REQUIRE((T + bt - 1) / bt <= max_blocks, CQ_ERR_INVALID, w + ": max_blocks too small");
  return CQ_OK;
}

static int launch_bounds(const sparse::BoundsArgs &A, cudaStream_t st, const char *what) {
  const int64_t grid = (int64_t)A.cv.B * A.cv.H * A.nb;
  CQ_REQUIRE(grid < (1LL << 31), CQ_ERR_INVALID, std::string(what) + ": grid too large");
  const int threads = (A.cv.D + 31) & ~31;
  sparse::block_bounds_kernel<<<(unsigned)grid, threads, 0, st>>>(A);
  return check_launch(what);
}

extern "C" int cq_block_bounds(const cq_paged_cache *cache, int64_t t0, int64_t T, int32_t block_tokens, int8_t *codes,
                               float *scales, int64_t max_blocks, void *stream) {
  int r = bounds_checks(cache, T, block_tokens, codes, scales, max_blocks, "cq_block_bounds");
  if (r) return r;
  CQ_REQUIRE(t0 >= 0 && t0 <= T, CQ_ERR_INVALID, "cq_block_bounds: t0 must lie in [0, T]");
  if (t0 == T) return CQ_OK;
  sparse::BoundsArgs A{make_view(*cache), t0, T, nullptr, 0, block_tokens, 0, codes, scales, max_blocks};
  A.nb = (int)((T - 1) / block_tokens - t0 / block_tokens + 1);
  return launch_bounds(A, (cudaStream_t)stream, "cq_block_bounds");
}

extern "C" int cq_block_bounds_at(const cq_paged_cache *cache, const int64_t *len_dev, int64_t max_len, int32_t S,
                                  int32_t block_tokens, int8_t *codes, float *scales, int64_t max_blocks,
                                  void *stream) {
  int r = bounds_checks(cache, max_len, block_tokens, codes, scales, max_blocks, "cq_block_bounds_at");
  if (r) return r;
  CQ_REQUIRE(len_dev && S >= 1 && S <= max_len, CQ_ERR_INVALID, "cq_block_bounds_at: bad length arguments");
  sparse::BoundsArgs A{make_view(*cache), 0, max_len, len_dev, S, block_tokens, 0, codes, scales, max_blocks};
  A.nb = (S + block_tokens - 2) / block_tokens + 1;  // the most blocks S tokens can touch
  return launch_bounds(A, (cudaStream_t)stream, "cq_block_bounds_at");
}

extern "C" int cq_block_bounds_read(const int8_t *codes, const float *scales, int64_t units, int64_t max_blocks,
                                    int64_t first, int64_t n, int32_t head_dim, float *out, void *stream) {
  CQ_REQUIRE(codes && scales && out, CQ_ERR_INVALID, "cq_block_bounds_read: null pointer");
  CQ_REQUIRE(units >= 1 && first >= 0 && n >= 0 && n <= max_blocks - first && head_dim >= 8 && head_dim <= 256,
             CQ_ERR_INVALID, "cq_block_bounds_read: bad sizes");
  if (n == 0) return CQ_OK;
  const int64_t grid = (units * n * 32 + 255) / 256;
  CQ_REQUIRE(grid < (1LL << 31), CQ_ERR_INVALID, "cq_block_bounds_read: grid too large");
  sparse::bounds_read_kernel<<<(unsigned)grid, 256, 0, (cudaStream_t)stream>>>(codes, scales, units, max_blocks, first,
                                                                              n, head_dim, out);
  return check_launch("cq_block_bounds_read");
}

static int select_sizes(int32_t batch, int32_t kv_heads, int32_t q_len, int64_t T, int32_t block_tokens,
                        size_t *bytes) {
  CQ_REQUIRE(batch >= 1 && kv_heads >= 1 && block_tokens >= 1, CQ_ERR_INVALID, "cq_block_select: bad sizes");
  CQ_REQUIRE(q_len >= 1 && q_len <= T, CQ_ERR_INVALID, "cq_block_select: need 1 <= q_len <= T");
  *bytes = (size_t)batch * kv_heads * q_len * ((T + block_tokens - 1) / block_tokens) * sizeof(float);
  return CQ_OK;
}

extern "C" int cq_block_select_workspace(int32_t batch, int32_t kv_heads, int32_t q_len, int64_t T,
                                         int32_t block_tokens, size_t *bytes) {
  CQ_REQUIRE(bytes, CQ_ERR_INVALID, "cq_block_select_workspace: bytes is null");
  return select_sizes(batch, kv_heads, q_len, T, block_tokens, bytes);
}

extern "C" int cq_block_select(const int8_t *codes, const float *scales, int64_t max_blocks, int32_t block_tokens,
                               int32_t batch, int32_t kv_heads, int32_t head_dim, int64_t T, const int64_t *len_dev,
                               const void *q, int q_dtype, int32_t n_q_heads, int32_t q_len, int64_t q_sb,
                               int64_t q_sh, int64_t q_sq, const int64_t *starts, int32_t first, int32_t recent,
                               int32_t top, int32_t *blocks, float *block_scores, void *workspace,
                               size_t workspace_bytes, void *stream) {
  size_t need = 0;
  int r = select_sizes(batch, kv_heads, q_len, T, block_tokens, &need);
  if (r) return r;
  CQ_REQUIRE(codes && scales && q && blocks, CQ_ERR_INVALID, "cq_block_select: null pointer");
  CQ_REQUIRE(head_dim >= 8 && head_dim <= 256 && head_dim % 8 == 0, CQ_ERR_UNSUPPORTED,
             "cq_block_select: head_dim must be a multiple of 8 in [8, 256]");
  CQ_REQUIRE(q_dtype == CQ_F16 || q_dtype == CQ_BF16, CQ_ERR_UNSUPPORTED, "cq_block_select: q dtype must be f16/bf16");
  CQ_REQUIRE(n_q_heads >= 1 && n_q_heads % kv_heads == 0, CQ_ERR_INVALID,
             "cq_block_select: n_q_heads must be a positive multiple of kv_heads");
  CQ_REQUIRE(first >= 0 && recent >= 0 && top >= 1 && first <= top && recent <= top - first, CQ_ERR_INVALID,
             "cq_block_select: need first + recent <= top");
  CQ_REQUIRE(top <= sparse::kMaxTop, CQ_ERR_UNSUPPORTED, "cq_block_select: top must be <= 4096");
  const int64_t n = (T + block_tokens - 1) / block_tokens;
  CQ_REQUIRE(n <= max_blocks && n < (1LL << 30), CQ_ERR_INVALID, "cq_block_select: T beyond the summarised blocks");
  CQ_REQUIRE(workspace && workspace_bytes >= need, CQ_ERR_WORKSPACE, "cq_block_select: workspace too small");
  sparse::SelectArgs A{codes,  scales, max_blocks, block_tokens, batch, kv_heads, head_dim, n_q_heads / kv_heads,
                       q_len,  T,      len_dev,    q,            q_dtype, q_sb,   q_sh,     q_sq,
                       starts, first,  recent,     top,          blocks,  block_scores,     n, (float *)workspace};
  const int64_t rows = (int64_t)batch * kv_heads * q_len, grid = (rows * n * 32 + 255) / 256;
  CQ_REQUIRE(grid < (1LL << 31), CQ_ERR_INVALID, "cq_block_select: grid too large");
  cudaStream_t st = (cudaStream_t)stream;
  sparse::block_score_kernel<<<(unsigned)grid, 256, 0, st>>>(A);
  r = check_launch("cq_block_select");
  if (r) return r;
  sparse::block_topk_kernel<<<(unsigned)rows, 256, 0, st>>>(A);
  return check_launch("cq_block_select");
}

static int sparse_checks(const cq_paged_cache *cache, int64_t T, int32_t n_q_heads, int32_t q_len, int32_t top,
                         int32_t bt) {
  int r = validate_cache(cache);
  if (r) return r;
  CQ_REQUIRE(n_q_heads >= 1 && n_q_heads % cache->kv_heads == 0, CQ_ERR_INVALID,
             "cq_sparse_attention: n_q_heads must be a positive multiple of kv_heads");
  CQ_REQUIRE(q_len >= 1 && q_len <= T, CQ_ERR_INVALID, "cq_sparse_attention: need 1 <= q_len <= T");
  CQ_REQUIRE((T + cache->page_tokens - 1) / cache->page_tokens <= cache->max_pages, CQ_ERR_INVALID,
             "cq_sparse_attention: T beyond mapped pages");
  CQ_REQUIRE(top >= 1 && bt >= 1, CQ_ERR_INVALID, "cq_sparse_attention: bad list length or block_tokens");
  CQ_REQUIRE(top <= sparse::kMaxTop, CQ_ERR_UNSUPPORTED, "cq_sparse_attention: at most 4096 blocks per list");
  return CQ_OK;
}

extern "C" int cq_sparse_attention_workspace(const cq_paged_cache *cache, int64_t T, int32_t n_q_heads, int32_t q_len,
                                             int32_t top, int32_t block_tokens, size_t *bytes) {
  int r = sparse_checks(cache, T, n_q_heads, q_len, top, block_tokens);
  if (r) return r;
  CQ_REQUIRE(bytes, CQ_ERR_INVALID, "cq_sparse_attention_workspace: bytes is null");
  if (sparse_fast_supported(*cache, n_q_heads, block_tokens)) {
    *bytes = 0;
    return CQ_OK;
  }
  const int64_t rows = (int64_t)cache->batch * n_q_heads * q_len;
  *bytes = sparse::generic_bytes(rows, sparse::pick_list_splits(rows, top), cache->head_dim);
  return CQ_OK;
}

extern "C" int cq_sparse_attention(const cq_paged_cache *cache, int64_t T, const int64_t *len_dev, const void *q,
                                   int q_dtype, int32_t n_q_heads, int32_t q_len, int64_t q_sb, int64_t q_sh,
                                   int64_t q_sq, float scale, const int64_t *starts, const int32_t *blocks,
                                   int32_t top, int32_t block_tokens, void *out, int out_dtype, float *lse_out,
                                   void *workspace, size_t workspace_bytes, void *stream) {
  int r = sparse_checks(cache, T, n_q_heads, q_len, top, block_tokens);
  if (r) return r;
  CQ_REQUIRE(q && blocks && out, CQ_ERR_INVALID, "cq_sparse_attention: null pointer");
  CQ_REQUIRE(q_dtype == CQ_F16 || q_dtype == CQ_BF16, CQ_ERR_UNSUPPORTED,
             "cq_sparse_attention: q dtype must be f16/bf16");
  CQ_REQUIRE(out_dtype == CQ_F16 || out_dtype == CQ_BF16 || out_dtype == CQ_F32, CQ_ERR_UNSUPPORTED,
             "cq_sparse_attention: bad out dtype");
  const int64_t rows = (int64_t)cache->batch * n_q_heads * q_len;
  if (sparse_fast_supported(*cache, n_q_heads, block_tokens))
    return run_sparse_fast(*cache, T, len_dev, q, q_dtype, n_q_heads, q_len, q_sb, q_sh, q_sq, scale, starts, blocks,
                           top, block_tokens, out, out_dtype, lse_out, (cudaStream_t)stream);
  const int splits = sparse::pick_list_splits(rows, top), D = cache->head_dim;
  CQ_REQUIRE(workspace && workspace_bytes >= sparse::generic_bytes(rows, splits, D), CQ_ERR_WORKSPACE,
             "cq_sparse_attention: workspace too small");
  CQ_REQUIRE(rows * splits < (1LL << 31), CQ_ERR_INVALID, "cq_sparse_attention: grid too large");
  float *o = (float *)workspace, *m = o + rows * splits * D, *l = m + rows * splits;
  sparse::SparseArgs A{make_view(*cache), q,     q_dtype, n_q_heads, q_len, top,    block_tokens, splits, q_sb, q_sh, q_sq,
                       scale,             T,     len_dev, starts,    blocks, m,     l,            o};
  cudaStream_t st = (cudaStream_t)stream;
  sparse::sparse_generic_kernel<<<(unsigned)(rows * splits), sparse::kGenWarps * 32, 0, st>>>(A);
  r = check_launch("cq_sparse_attention");
  if (r) return r;
  return launch_split_combine(m, l, o, rows, splits, D, out, out_dtype, lse_out, st);
}
