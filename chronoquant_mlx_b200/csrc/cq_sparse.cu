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
#include <string>
#include <type_traits>

#include "cq_launch.cuh"
#include "cq_prefill.cuh"
#include "cq_ptx.cuh"
#include "cq_sparse.cuh"

namespace cq {
namespace sparse {

__device__ int g_sparse_error;
__device__ void set_length_error() { atomicExch(&g_sparse_error, ERR_LENGTH); }

// ---------------------------------------------------------------------------
// bounds of any layout: one CTA per (sequence, kv-head, block), a thread per
// channel that walks the tokens in turn, so bound by the latency of its loads
// (8 x 16384 tokens of 8 heads of 96: 941 us; heads of 128 take 28 in the next one)
// ---------------------------------------------------------------------------
struct BoundsArgs {
  CacheView cv;
  int64_t t0, T;            // blocks of tokens t0 .. T-1
  const int64_t *len_dev;   // else: of the last S tokens of *len_dev
  int S, bt, nb;            // nb: blocks per unit in the grid
  int64_t j0;               // the first of them, without len_dev
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

// The least whole number c with c * s >= x (s > 0, |x| <= 126 s up to rounding;
// r about 1 / s): rint(x * r) is one of the two whole numbers next to x / s, and
// the exact sign of x - c * s tells which.
__device__ __forceinline__ float ceil_code(float x, float s, float r) {
  const float c = rintf(x * r);
  return fmaf(-c, s, x) > 0.f ? c + 1.f : c;
}

// One channel's codes from its range, in the low bytes (lower, upper); s: the
// block's scale (max|x| / 126), r about 1 / s, both 0 where every key is 0.
__device__ __forceinline__ int2 range_codes(float lo, float hi, float s, float r) {
  const float h = ceil_code(hi, s, r), l = -ceil_code(-lo, s, r);
  return make_int2((int)fminf(fmaxf(l, -127.f), 127.f), (int)fminf(fmaxf(h, -127.f), 127.f));
}

__global__ void __launch_bounds__(256) block_bounds_kernel(BoundsArgs A) {
  __shared__ float s_red[8];
  ptx::grid_dependency_wait();
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
  if (d < cv.D) {
    const int2 c = range_codes(lo, hi, s, s > 0.f ? 1.f / s : 0.f);
    int8_t *codes = A.codes + row * 2 * cv.D + d;
    codes[0] = (int8_t)c.x;
    codes[cv.D] = (int8_t)c.y;
  }
  if (threadIdx.x == 0) A.scales[row] = s;
}

// The same for the common layouts: head sizes D of 64, 128 or 256, K codes in
// natural order with token-indexed scales, rows 4-byte aligned, strides that are
// a multiple of the rows a warp takes at once.  A warp per block: a lane holds
// one code word (8 channels) of a row, D / 8 lanes a row, so 256 / D tokens at
// a time.  Keys of one anchor are anchor + p, p = code * scale rounded to fp16;
// rounding the sum keeps the order of p, so the packed minimum and maximum run
// over p and the anchor is added once at the end.  The kernel is bound by
// instructions, the ALU's first (half rate: mask, half a shift, minimum and
// maximum of a code pair): with one word a lane the lanes' meeting at the end,
// the anchors and the addresses cost a third of what they cost with four (2012
// instructions per 64 tokens of two anchors then).  8 x 16384 tokens of 8 heads
// of 128 (78 MB) take 33 us with their ranges read back.  An I-frame's scale slot is
// 0, so whatever its row reads (the row before it, inside the chunk block; the
// chunk's first token reads row 0) gives p = 0, the anchor itself.

// p of a code word's 4 pairs (channels k and k + 4) into the running minimum and maximum.
__device__ __forceinline__ void range_of_word(uint32_t word, __half2 scale, __half2 (&lo)[4], __half2 (&hi)[4]) {
  const __half2 m1032 = __float2half2_rn(-1032.f), sixteenth = __float2half2_rn(0.0625f), m72 = __float2half2_rn(-72.f);
  const uint32_t w8 = word >> 8;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    // nibbles k and k + 4 as 1024 + n, or as 1024 + 16 n, then the codes n - 8, exactly
    const uint32_t v = ptx::lop3_and_or(k < 2 ? word : w8, k & 1 ? 0x00f000f0u : 0x000f000fu, 0x64006400u);
    const __half2 code = k & 1 ? __hfma2(ptx::u2h2(v), sixteenth, m72) : __hadd2_rn(ptx::u2h2(v), m1032);
    const __half2 p = __hmul2_rn(code, scale);
    lo[k] = __hmin2(lo[k], p);  // a NaN is left out
    hi[k] = __hmax2(hi[k], p);
  }
}

// Positions are stepped from anchor to anchor (divisions for each: 36 us); with
// nine or ten CTAs an SM, or half the loads in flight: 34, 37 and 39 us.
template <int D>
__global__ void __launch_bounds__(128) block_bounds_rows_kernel(BoundsArgs A) {
  constexpr int W = D / 8, RPI = 32 / W;  // words (lanes) per row, rows at once
  constexpr int UN = 8;                   // steps whose loads are in flight
  const int lane = threadIdx.x & 31;
  ptx::grid_dependency_wait();
  const CacheView &cv = A.cv;
  const CompView &c = cv.c[0];
  // positions in 32 bits (the launch keeps them there)
  unsigned T = (unsigned)A.T, j = (unsigned)A.j0;
  if (A.len_dev) {
    T = (unsigned)launch_length(A.T, A.len_dev, A.S);
    if (T == 0) {
      if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) set_length_error();
      return;
    }
    j = (T - (unsigned)A.S) / (unsigned)A.bt;
  }
  const unsigned wi = blockIdx.x * 4 + (threadIdx.x >> 5), unit = blockIdx.y;
  if (wi >= (unsigned)A.nb) return;
  j += wi;
  if (j * (unsigned)A.bt >= T) return;
  const int ta = (int)(j * (unsigned)A.bt), tb = (int)min(T, (unsigned)(ta + A.bt));
  const int b = (int)(unit / (unsigned)cv.H), h = (int)(unit - (unsigned)b * (unsigned)cv.H);
  const int row = lane / W, word = lane % W;  // which of the rows at once, which 8 channels
  const __half2 inf = __float2half2_rn(INFINITY), ninf = __float2half2_rn(-INFINITY);
  __half2 lo[4], hi[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) lo[k] = inf, hi[k] = ninf;

  const int ct = c.pc + c.ac;  // tokens per chunk
  // one anchor's tokens at a time: they lie in one chunk of one page
  int lp = (int)((unsigned)ta / (unsigned)cv.P), tl = ta - lp * cv.P;          // page, position in it
  int jc = (int)((unsigned)tl / (unsigned)ct), x0 = tl - jc * ct;              // chunk, position in it
  int xa = (int)((unsigned)x0 / (unsigned)c.stride);                           // its anchor in the chunk
  for (int t = ta;;) {
    const int n = min(tb - t, (xa + 1) * c.stride - x0);
    const int64_t ph = page_of(cv, b, lp) * cv.H + h;  // looked up again rather than held: registers are short
    const uint4 an = *(const uint4 *)(c.kf + ph * c.kf_hs + jc * c.kf_cs + xa * D + word * 8);
    const int i0 = x0 - xa - 1 + row;  // this lane's first code row
    const uint32_t *crow = c.codes + ph * c.cd_hs + jc * c.cd_cs + i0 * W + word;
    const __half *sc = c.scales + ph * c.sc_hs + jc * c.sc_cs + x0 + row;
    __half2 plo[4], phi[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) plo[k] = inf, phi[k] = ninf;
    for (int r = 0; r < n; r += UN * RPI) {
      uint32_t code[UN];
      __half s1[UN];
      if (r + UN * RPI <= n) {
#pragma unroll
        for (int u = 0; u < UN; ++u) {
          code[u] = u == 0 && i0 + r < 0 ? 0u : crow[(r + u * RPI) * W];
          s1[u] = sc[r + u * RPI];
        }
      } else {  // rows past the end give NaN, which is left out
#pragma unroll
        for (int u = 0; u < UN; ++u) {
          const bool in = r + u * RPI + row < n;
          code[u] = !in || i0 + r + u * RPI < 0 ? 0u : crow[(r + u * RPI) * W];
          s1[u] = in ? sc[r + u * RPI] : __ushort_as_half(0x7fffu);
        }
      }
#pragma unroll
      for (int u = 0; u < UN; ++u) range_of_word(code[u], __half2half2(s1[u]), plo, phi);
    }
    const uint32_t p[4] = {an.x, an.y, an.z, an.w};  // channels (0,1) (2,3) (4,5) (6,7)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t pr = __byte_perm(p[k >> 1], p[2 + (k >> 1)], (k & 1) ? 0x7632u : 0x5410u);
      lo[k] = __hmin2(lo[k], __hadd2_rn(ptx::u2h2(pr), plo[k]));
      hi[k] = __hmax2(hi[k], __hadd2_rn(ptx::u2h2(pr), phi[k]));
    }
    t += n;
    if (t >= tb) break;
    ++xa;  // an anchor's last token was passed: the next anchor, chunk or page
    x0 += n;
    tl += n;
    if (x0 == ct) x0 = xa = 0, ++jc;
    if (tl == cv.P) tl = jc = 0, ++lp;
  }
  // lanes of the same channels: rows meet by halves, each keeping half of its pairs, until a lane holds 4 / RPI pairs
  int k0 = 0;  // first pair this lane still holds
  auto meet = [&](auto pairs, int o) {
    constexpr int m = decltype(pairs)::value / 2;
    const bool up = lane & o;
#pragma unroll
    for (int k = 0; k < m; ++k) {
      const __half2 la = lo[k], lb = lo[k + m], ha = hi[k], hb = hi[k + m];
      lo[k] = __hmin2(up ? lb : la, __shfl_xor_sync(0xffffffffu, up ? la : lb, o));
      hi[k] = __hmax2(up ? hb : ha, __shfl_xor_sync(0xffffffffu, up ? ha : hb, o));
    }
    if (up) k0 += m;
  };
  if constexpr (RPI >= 2) meet(std::integral_constant<int, 4>(), 16);
  if constexpr (RPI >= 4) meet(std::integral_constant<int, 2>(), 8);
  constexpr int NP = 4 / RPI;  // pairs a lane ends with
  float l[2 * NP], u[2 * NP], amax = 0.f;
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    const float2 x = __half22float2(lo[k]), y = __half22float2(hi[k]);
    const float lv[2] = {x.x, x.y}, uv[2] = {y.x, y.y};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float p = lv[e], q = uv[e];
      if (p > q) p = q = 0.f;  // no value at all
      p = fminf(fmaxf(p, -65504.f), 65504.f);
      q = fminf(fmaxf(q, -65504.f), 65504.f);
      l[2 * k + e] = p;
      u[2 * k + e] = q;
      amax = fmaxf(amax, fmaxf(fabsf(p), fabsf(q)));
    }
  }
  amax = warp_max(amax);
  const float s = __fdiv_rn(amax, 126.f);
  const float r = s > 0.f ? 1.f / s : 0.f;
  const int64_t at = (int64_t)unit * A.max_blocks + j;
  int8_t *codes = A.codes + at * 2 * D + word * 8 + k0;
#pragma unroll
  for (int e = 0; e < 2; ++e) {  // NP neighbouring channels from k0 on, and from k0 + 4 on
    uint32_t lw = 0, uw = 0;
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int2 q = range_codes(l[2 * k + e], u[2 * k + e], s, r);
      lw |= ((uint32_t)q.x & 255u) << (8 * k);
      uw |= ((uint32_t)q.y & 255u) << (8 * k);
    }
    using Store = typename std::conditional<NP == 4, uint32_t, typename std::conditional<NP == 2, uint16_t, uint8_t>::type>::type;
    *(Store *)(codes + 4 * e) = (Store)lw;
    *(Store *)(codes + D + 4 * e) = (Store)uw;
  }
  if (lane == 0) A.scales[at] = s;
}

// out [units][n][2][D] fp32 = code * scale of blocks first .. first + n - 1;
// a warp per block, four codes a lane at a time (2D is a multiple of 4).
__global__ void __launch_bounds__(256) bounds_read_kernel(const int8_t *codes, const float *scales, int64_t units,
                                                          int64_t max_blocks, int64_t first, int64_t n, int D,
                                                          float *out) {
  ptx::grid_dependency_wait();
  const int64_t row = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (row >= units * n) return;
  const int64_t u = row / n, j = first + (row - u * n);
  const char4 *c = (const char4 *)(codes + (u * max_blocks + j) * 2 * D);
  const float s = scales[u * max_blocks + j];
  float4 *o = (float4 *)(out + row * 2 * D);
  for (int i = threadIdx.x & 31; i < D / 2; i += 32) {
    const char4 v = c[i];
    o[i] = make_float4((float)v.x * s, (float)v.y * s, (float)v.z * s, (float)v.w * s);
  }
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
  int64_t n, ns;  // blocks of T, stride of a score row (a multiple of 8)
  float *score;   // [units][q_len][ns]
};

// One row of query codes: values x (finite, in the fp16 range) of amax, code rint(x * (127 / amax)).
struct QueryScale {
  float r, s;
  __device__ explicit QueryScale(float amax) {
    const bool zero = amax < kTinyQuery;
    r = zero ? 0.f : __fdiv_rn(127.f, amax);
    s = zero ? 0.f : __fdiv_rn(amax, 127.f);
  }
  __device__ int code(float x) const { return (int)rintf(__fmul_rn(x, r)); }
};

// D(16x8 s32) += A(16x32 s8, row) * B(32x8 s8, col)
__device__ __forceinline__ void mma_s8_16832(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Scores on the tensor cores (head sizes of KS * 32, groups of at most 16).
// Rows of the product are (query token, head) pairs, GP = the group rounded up
// to a power of two; columns are blocks; the sum runs over 2D codes, a query
// row holding [min(q8, 0) | max(q8, 0)] against a block's [lower | upper] codes.
// A lane loads 16 bytes of a block at a time; the order of the sum's terms is
// permuted alike in both operands, so these are two steps' B fragments as they
// come.  A CTA quantises `tiles` row tiles into shared memory once (rows 64
// bytes apart modulo 128: no bank conflicts), then each warp takes columns in
// `passes`, keeping two column tiles' codes in registers over the rows.  The
// maximum over a group's heads goes by halves: each exchange also halves the
// values a lane holds, so every lane ends with its own ones to store.  Bound by
// the instructions around the products, not by the tensor pipe: a row tile against
// 16 blocks is about 200, 16 of them products and 8 operand loads, the rest scaling
// and the heads' maximum across lanes, and 14 warps an SM issue in less than half
// of the slots.  2048 rows x 1024 blocks x 256 codes x 8 units take 27
// us (7.5 us of products); two row tiles at once 29, half the row tiles a CTA 34,
// and with the codes as fp16, whose fragments cost conversions, 47 us.  One launch
// that also lists, with the scores in shared memory, took 10 us more there than
// this kernel and the next: too few warps fit beside the scores.
constexpr int kScoreWarps = 8, kScoreCols = 16;  // blocks per warp and pass

// Query rows [0, rows) of a unit from token i0 on into shared memory, by WARPS
// warps.  A lane holds KS channels next to each other: one load where the rows are
// aligned for it, one store each for the two halves of a code row.  The rows
// behind the group's heads get the scale NaN.
template <int KS, int GP, int WARPS>
__device__ __forceinline__ void quantise_rows(const SelectArgs &A, unsigned unit, int i0, int rows, unsigned char *s_a,
                                              float *s_sg) {
  constexpr int D = KS * 32, STR = 2 * D + 64, UN = WARPS > 8 ? 1 : 4;  // rows whose loads are in flight
  constexpr bool VEC = KS != 3;
  using Raw = typename std::conditional<KS == 8, uint4, typename std::conditional<KS == 4, uint2, uint32_t>::type>::type;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = (int)(unit / (unsigned)A.H), h = (int)(unit - (unsigned)b * (unsigned)A.H);
  const bool wide = VEC && ((((uintptr_t)A.q) & (2 * KS - 1)) | ((uint64_t)(A.q_sb | A.q_sh | A.q_sq) & (KS - 1))) == 0;
  for (int r0 = warp; r0 < rows; r0 += UN * WARPS) {
    float x[UN][KS];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int r = r0 + u * WARPS, i = i0 + r / GP, hd = r & (GP - 1);
      const bool real = r < rows && i < A.q_len && hd < A.G;
      const int64_t at = b * A.q_sb + (int64_t)(h * A.G + hd) * A.q_sh + (int64_t)i * A.q_sq + lane * KS;
      if (VEC && wide) {
        Raw w = {};
        if (real) w = *(const Raw *)((const uint16_t *)A.q + at);
        const uint32_t *p = (const uint32_t *)&w;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const uint16_t e = (uint16_t)(p[k / 2] >> (k & 1 ? 16 : 0));
          x[u][k] = A.q_dtype == CQ_BF16 ? __uint_as_float((uint32_t)e << 16) : __half2float(__ushort_as_half(e));
        }
      } else {
#pragma unroll
        for (int k = 0; k < KS; ++k) x[u][k] = real ? load_as_float(A.q, at + k, A.q_dtype) : 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int r = r0 + u * WARPS;
      if (r >= rows) break;
      float amax = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        x[u][k] = finite_query(x[u][k]);
        amax = fmaxf(amax, fabsf(x[u][k]));
      }
      const QueryScale qs(warp_max(amax));
      int8_t *row = (int8_t *)s_a + r * STR + lane * KS;
      uint32_t lo[(KS + 3) / 4] = {}, hi[(KS + 3) / 4] = {};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int c = qs.code(x[u][k]);
        lo[k / 4] |= ((uint32_t)min(c, 0) & 255u) << (8 * (k & 3));
        hi[k / 4] |= (uint32_t)max(c, 0) << (8 * (k & 3));
      }
      if constexpr (KS == 2) {
        *(uint16_t *)row = (uint16_t)lo[0];
        *(uint16_t *)(row + D) = (uint16_t)hi[0];
      } else if constexpr (KS == 3) {
#pragma unroll
        for (int k = 0; k < 3; ++k) row[k] = (int8_t)(lo[0] >> (8 * k)), row[D + k] = (int8_t)(hi[0] >> (8 * k));
      } else {
#pragma unroll
        for (int k = 0; k < KS / 4; ++k) ((uint32_t *)row)[k] = lo[k], ((uint32_t *)(row + D))[k] = hi[k];
      }
      if (lane == 0) s_sg[r] = (r & (GP - 1)) < A.G ? qs.s : __int_as_float(0x7fffffff);
    }
  }
}

// A warp's two column tiles: the B fragments of blocks j0 .. j0 + 15 and their scales.
template <int KS>
struct BlockCodes {
  uint4 bf[2][KS];
  float sj[2][2];
  __device__ __forceinline__ BlockCodes(const SelectArgs &A, unsigned unit, int j0) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, last = (int)A.n - 1;
    const int8_t *codes = A.codes + (int64_t)unit * A.max_blocks * (2 * KS * 32);
    const float *scales = A.scales + (int64_t)unit * A.max_blocks;
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
      const int8_t *src = codes + (int64_t)min(j0 + nb * 8 + g, last) * (2 * KS * 32) + 16 * t;
#pragma unroll
      for (int k = 0; k < KS; ++k) bf[nb][k] = *(const uint4 *)(src + 64 * k);
#pragma unroll
      for (int e = 0; e < 2; ++e) sj[nb][e] = scales[min(j0 + nb * 8 + 2 * t + e, last)];
    }
  }
};

// Scores of one row tile (its codes at a_tile, its scales at sg_tile; its first
// token is i) against blocks j0 .. j0 + 15: token tok's go to dst[tok * ns].
template <int KS, int GP>
__device__ __forceinline__ void score_tile(const SelectArgs &A, const BlockCodes<KS> &f, const unsigned char *a_tile,
                                           const float *sg_tile, int i, int j0, float *dst) {
  constexpr int STR = 2 * KS * 32 + 64;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  int acc[2][4] = {};
  const unsigned char *a = a_tile + g * STR + 16 * t;
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    const uint4 x = *(const uint4 *)(a + 64 * k), y = *(const uint4 *)(a + 8 * STR + 64 * k);
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
      mma_s8_16832(acc[nb], x.x, y.x, x.y, y.y, f.bf[nb][k].x, f.bf[nb][k].y);
      mma_s8_16832(acc[nb], x.z, y.z, x.w, y.w, f.bf[nb][k].z, f.bf[nb][k].w);
    }
  }
  const float sg0 = sg_tile[g], sg1 = sg_tile[g + 8];
  // v[column tile][row half][column]: scores of rows g and g + 8
  float v[2][2][2];
#pragma unroll
  for (int nb = 0; nb < 2; ++nb)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float x = __fmul_rn(__fmul_rn(sg0, f.sj[nb][e]), (float)acc[nb][e]);
      const float y = __fmul_rn(__fmul_rn(sg1, f.sj[nb][e]), (float)acc[nb][2 + e]);
      v[nb][0][e] = x;  // NaN in the rows behind the group, which the maximum leaves out
      v[nb][1][e] = y;
    }
  auto swap_max = [&](float &keep, float give, int o) { keep = fmaxf(keep, __shfl_xor_sync(0xffffffffu, give, o)); };
  int nb0 = 0, hf0 = 0;  // which of the values this lane holds
  if constexpr (GP == 16) {
#pragma unroll
    for (int nb = 0; nb < 2; ++nb)
#pragma unroll
      for (int e = 0; e < 2; ++e) v[nb][0][e] = fmaxf(v[nb][0][e], v[nb][1][e]);
  }
  if constexpr (GP >= 2) {  // heads in lane bit 2: keep one column tile
    nb0 = g & 1;
#pragma unroll
    for (int hf = 0; hf < (GP == 16 ? 1 : 2); ++hf)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float a0 = v[0][hf][e], a1 = v[1][hf][e];
        v[0][hf][e] = nb0 ? a1 : a0;
        swap_max(v[0][hf][e], nb0 ? a0 : a1, 4);
      }
  }
  if constexpr (GP == 4 || GP == 8) {  // heads in lane bit 3: keep one row half
    hf0 = (g >> 1) & 1;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float a0 = v[0][0][e], a1 = v[0][1][e];
      v[0][0][e] = hf0 ? a1 : a0;
      swap_max(v[0][0][e], hf0 ? a0 : a1, 8);
    }
  }
  if constexpr (GP == 16)
#pragma unroll
    for (int e = 0; e < 2; ++e) v[0][0][e] = fmaxf(v[0][0][e], __shfl_xor_sync(0xffffffffu, v[0][0][e], 8));
  if constexpr (GP >= 8)  // heads in lane bit 4
#pragma unroll
    for (int e = 0; e < 2; ++e) v[0][0][e] = fmaxf(v[0][0][e], __shfl_xor_sync(0xffffffffu, v[0][0][e], 16));
  // token (in the tile) of the lane's row g, and of row g + 8: 8 / GP further on
  const int ta = g / GP;
  constexpr int NBV = GP >= 2 ? 1 : 2, HFV = GP == 1 || GP == 2 ? 2 : 1;
#pragma unroll
  for (int nb = 0; nb < NBV; ++nb)
#pragma unroll
    for (int hf = 0; hf < HFV; ++hf) {
      const int tok = ta + (HFV == 2 ? hf : hf0) * (8 / GP), col = (NBV == 2 ? nb : nb0) * 8 + 2 * t;
      bool mine = i + tok < A.q_len && j0 + col < (int)A.ns;
      if (GP >= 8) mine = mine && !(g & 4);
      if (GP == 16) mine = mine && !(g & 2);
      if (mine)  // -0 becomes +0: equal scores have equal keys
        *(float2 *)(dst + tok * A.ns + col) = make_float2(__fadd_rn(v[nb][hf][0], 0.f), __fadd_rn(v[nb][hf][1], 0.f));
    }
}

template <int KS, int GP>
__global__ void __launch_bounds__(kScoreWarps * 32) block_score_mma_kernel(SelectArgs A, int tiles, int passes) {
  constexpr int STR = 2 * KS * 32 + 64, TPT = 16 / GP;  // query tokens per row tile
  extern __shared__ __align__(16) unsigned char s_a[];  // [tiles * 16][STR], then fp32 [tiles * 16]
  float *s_sg = (float *)(s_a + tiles * 16 * STR);
  const unsigned unit = blockIdx.z;
  const int i0 = blockIdx.y * tiles * TPT;
  ptx::grid_dependency_wait();
  const int64_t T = launch_length(A.T, A.len_dev, A.q_len);
  if (T == 0) return;
  quantise_rows<KS, GP, kScoreWarps>(A, unit, i0, tiles * 16, s_a, s_sg);
  __syncthreads();
  // the last block any of this CTA's tokens sees
  const int i_last = min(A.q_len, i0 + tiles * TPT) - 1;
  const int j_end = (int)min((unsigned)A.n, (unsigned)(T - A.q_len + i_last) / (unsigned)A.bt + 1u);  // T below 2^31
  const int real_tiles = (i_last - i0) / TPT + 1;
  for (int pass = 0; pass < passes; ++pass) {
    const int j0 = (int)((blockIdx.x * passes + pass) * kScoreWarps + (threadIdx.x >> 5)) * kScoreCols;
    if (j0 >= j_end) break;
    const BlockCodes<KS> f(A, unit, j0);
    float *dst = A.score + ((int64_t)unit * A.q_len + i0) * A.ns + j0;  // of this row tile's first token
    for (int rt = 0; rt < real_tiles; ++rt, dst += TPT * A.ns)
      score_tile<KS, GP>(A, f, s_a + rt * 16 * STR, s_sg + rt * 16, i0 + rt * TPT, j0, dst);
  }
}

// Every other shape: one warp per (unit, query token, block).
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
    const QueryScale qs(warp_max(amax));
    int dot = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int d = lane + 32 * k;
      if (d < A.D) {
        const int q8 = qs.code(x[k]);
        dot += q8 * (int)(q8 > 0 ? c[A.D + d] : c[d]);
      }
    }
    dot = __reduce_add_sync(0xffffffffu, dot);
    best = fmaxf(best, __fmul_rn(__fmul_rn(qs.s, sj), (float)dot));
  }
  if (lane == 0) A.score[row * A.ns + j] = __fadd_rn(best, 0.f);  // -0 becomes +0: equal scores have equal keys
}

// The `top` best visible blocks of a (unit, query token) row with every key in a
// register: W warps, each thread with the keys of KPT blocks next to each other.
// W is a trade of one row's time against the number of rows at once: of 4096 rows
// of 512, 1024, 2048 and 4096 blocks, one warp a row takes 7.8, 11.7 and 19.4 us,
// up to four 11.5, 14.5, 19.4 and 31.7, up to 32 with eight keys a thread 24 and
// 44 us for the last two; of 128 rows
// of 1024 one warp a row takes 5.6, eight of four keys a thread 4.2 us.
// First a threshold is guessed that some more than `top` keys reach, from the
// scores' mean and deviation: one count settles it for scores that look normal,
// where a search bit by bit takes a dozen (512 queries x 1024 blocks x 8 units, 32
// of each: 26 us without, 21 us with it).  If four guesses miss, the threshold key
// is found from the highest bit on which the row's keys differ: with up to four
// warps bit by bit (count the keys that reach a candidate), with more of them,
// whose meetings cost more, eight bits at a time by a histogram of the keys still
// in question.  As soon as no more than kShort keys reach the threshold so far,
// those are gathered in index order in shared memory, and one warp goes on with
// them alone, two bits at a time (ranking them against each other instead took 3
// us more).  Where that never happens (long lists, many equal keys) the search
// runs to the last bit.  The list is written in index order, of equal keys the
// lowest indexes.  Keys of neighbouring blocks in a thread make the positions a sum
// over threads (keys dealt out in turn, with a count per warp and turn: 21 us,
// this: 15 us).
constexpr int kShort = 128;

enum class Warps { ONE, FEW, MANY };  // a row's warps: one, up to four, up to 32

template <Warps N>
struct TopkShared {
  uint32_t key[kShort];
  int idx[kShort];
  int hist[N == Warps::MANY ? 256 : 1];
  int cnt[4];
  __align__(16) int pre[N == Warps::ONE ? 4 : 128];  // four a warp
};

// Query token i of a unit with its scores at `score` (16-byte aligned), by W
// warps (named barrier 1), of which this is number `warp`.
template <int KPT, Warps NW>
__device__ __forceinline__ void topk_row(const SelectArgs &A, int64_t T, unsigned unit, int i, const float *score,
                                         int n_warps, int warp, TopkShared<NW> &sh) {
  constexpr bool HIST = NW == Warps::MANY;
  const int W = NW == Warps::ONE ? 1 : n_warps;
  uint32_t *s_key = sh.key;
  int *s_idx = sh.idx, *s_hist = sh.hist, *s_cnt = sh.cnt, *s_pre = sh.pre;
  const int lane = threadIdx.x & 31;
  auto meet = [&]() {
    if (NW == Warps::ONE) __syncwarp();
    else ptx::named_barrier_sync(1, W * 32);
  };
  // 32-bit positions (the launch keeps T there): a 64-bit division takes a hundred instructions
  const unsigned bt = (unsigned)A.bt, p = (unsigned)(T - A.q_len) + (unsigned)i;
  int fb = 0, lb = (int)(p / bt);  // the blocks this token may see
  if (A.starts) {
    const int b = (int)(unit / (unsigned)A.H);
    const unsigned st = (unsigned)min(first_token(A.starts, b), (int64_t)INT32_MAX);
    fb = (int)(st / bt);
    if (st > p) lb = fb - 1;
  }
  const int nv = lb - fb + 1;
  const int64_t row = (int64_t)unit * A.q_len + i;
  int32_t *out = A.blocks + row * A.top;
  float *out_s = A.block_scores ? A.block_scores + row * A.top : nullptr;
  const int tid = warp * 32 + lane, step = W * 32;
  for (int k = min(nv, A.top) + tid; k < A.top; k += step) {
    out[k] = -1;
    if (out_s) out_s[k] = -INFINITY;
  }
  uint32_t key[KPT];  // of blocks j0 .. j0 + KPT - 1; 0: no block (visible ones are above it)
  uint32_t all_or = 0, all_and = 0xffffffffu;
  float s1 = 0.f, s2 = 0.f;  // sums of the scores that compete and of their squares
  const int j0 = tid * KPT;
  {
    float4 v[KPT / 4];
#pragma unroll
    for (int k = 0; k < KPT / 4; ++k)
      v[k] = j0 + 4 * k < (int)A.ns ? ((const float4 *)score)[(j0 >> 2) + k] : make_float4(0.f, 0.f, 0.f, 0.f);
    const unsigned rivals = (unsigned)max(nv - A.first - A.recent, 0);
#pragma unroll
    for (int k = 0; k < KPT; ++k) {
      const float x = (&v[k / 4].x)[k % 4];
      const int at = j0 + k - fb;
      key[k] = (unsigned)at < (unsigned)nv ? 0xffffffffu : 0u;
      if ((unsigned)(at - A.first) < rivals) {
        key[k] = order_key(x);
        all_or |= key[k];
        all_and &= key[k];
        s1 += x;
        s2 = fmaf(x, x, s2);
      }
    }
  }
  uint32_t thr = 1;   // keys at or above it are taken, those equal to it from the lowest index on
  uint32_t from = 1;  // a bound below it, at which the gathered keys begin
  int reach = nv;     // keys that reach thr, or from
  int bit = -1;
  if (nv > A.top) {
    // the bits above the highest differing one are those of every key that is not forced
    all_or = __reduce_or_sync(0xffffffffu, all_or);
    all_and = __reduce_and_sync(0xffffffffu, all_and);
    int above = A.first + A.recent;  // keys above those in question (all of them visible: nv > top)
    // the rank at which a guessed threshold aims: behind the last one taken, within what can be gathered
    const float rank = 1.25f * (float)(A.top - above) + 8.f, rivals = (float)(nv - above);
    const bool guess = nv > kShort && rank + (float)above <= 0.9f * kShort && rivals >= 2.f * rank;
    if (guess) s1 = warp_sum(s1), s2 = warp_sum(s2);
    if (W > 1) {
      if (lane == 0) {
        s_pre[4 * warp] = (int)all_or, s_pre[4 * warp + 1] = (int)all_and;
        s_pre[4 * warp + 2] = __float_as_int(s1), s_pre[4 * warp + 3] = __float_as_int(s2);
      }
      meet();
      const int4 of = lane < W ? ((const int4 *)s_pre)[lane] : make_int4(0, -1, 0, 0);
      all_or = __reduce_or_sync(0xffffffffu, (uint32_t)of.x);
      all_and = __reduce_and_sync(0xffffffffu, (uint32_t)of.y);
      if (guess) s1 = warp_sum(__int_as_float(of.z)), s2 = warp_sum(__int_as_float(of.w));
      meet();  // s_pre is written again below
    }
    const uint32_t differ = all_or & ~all_and;  // first + recent <= top < nv: some key is not forced
    bit = differ ? 31 - __clz(differ) : -1;
    thr = bit < 0 ? all_and : all_and & ~((2u << bit) - 1u);
    const bool shorten = A.top <= kShort;
    if (above == A.top) thr = 0xffffffffu, reach = A.top, bit = -1;  // the forced blocks fill the list
    // The threshold guessed: where a normal distribution of these scores' mean and deviation has `rank` of them
    // (quantile by Abramowitz and Stegun 26.2.22), moved by half a deviation while too few or too many reach it.
    if (guess && bit >= 0) {
      const float per = __fdividef(1.f, rivals), mean = s1 * per, var = fmaxf(s2 * per - mean * mean, 1e-30f);
      const float sd = var * rsqrtf(var), w = 2.f * __logf(rivals * __fdividef(1.f, rank)), u = w * rsqrtf(w);
      float z = u - __fdividef(2.30753f + 0.27061f * u, 1.f + u * (0.99229f + 0.04481f * u));
      for (int tries = 0; tries < 4; ++tries) {
        const uint32_t cand = max(order_key(fmaf(z, sd, mean)), 1u);
        int c = 0;
#pragma unroll
        for (int k = 0; k < KPT; ++k) c += key[k] >= cand;
        c = __reduce_add_sync(0xffffffffu, c);
        if (W > 1) {
          if (lane == 0) s_pre[(tries & 1) * 32 + warp] = c;
          meet();
          c = __reduce_add_sync(0xffffffffu, lane < W ? s_pre[(tries & 1) * 32 + lane] : 0);
        }
        if (c >= A.top && c <= kShort) {
          from = cand;
          reach = c;
          break;
        }
        z += c < A.top ? -0.5f : 0.5f;
      }
      if (W > 1) meet();  // s_pre is written again below
    }
    if (!HIST || W <= 4) {
      int par = 0;
      for (; bit >= 0 && reach != A.top && !(shorten && reach <= kShort); --bit) {
        const uint32_t cand = thr | (1u << bit);
        int c = 0;
#pragma unroll
        for (int k = 0; k < KPT; ++k) c += key[k] >= cand;
        c = __reduce_add_sync(0xffffffffu, c);
        if (W > 1) {
          if (lane == 0) s_pre[par * 4 + warp] = c;
          meet();
          c = __reduce_add_sync(0xffffffffu, lane < W ? s_pre[par * 4 + lane] : 0);
          par ^= 1;
        }
        if (c >= A.top) thr = cand, reach = c;
      }
      if (W > 1) meet();  // s_pre is written again below
    }
    while (HIST && W > 4 && bit >= 0 && reach != A.top && !(shorten && reach <= kShort)) {
      const int shift = max(bit - 7, 0), bins = 2 << (bit - shift);  // up to 8 bits
      for (int k = tid; k < 256; k += step) s_hist[k] = 0;
      meet();
      const uint32_t prefix = bit >= 31 ? 0u : thr >> (bit + 1);
#pragma unroll
      for (int k = 0; k < KPT; ++k)
        if (key[k] != 0u && key[k] != 0xffffffffu && (bit >= 31 || key[k] >> (bit + 1) == prefix))
          atomicAdd(&s_hist[(key[k] >> shift) & (bins - 1)], 1);
      meet();
      if (warp == 0) {  // the highest bin that brings the count to `top`: lane l holds bins 8l .. 8l + 7
        int c[8], sum = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += c[e] = s_hist[lane * 8 + e];
        int from = sum;  // of this lane's bins and all above
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_down_sync(0xffffffffu, from, o);
          if (lane + o < 32) from += x;
        }
        int over = above + from - sum;  // keys above this lane's bins
        if (over < A.top && over + sum >= A.top) {  // one lane
          int e = 7;
          while (over + c[e] < A.top) over += c[e--];
          s_cnt[0] = lane * 8 + e;
          s_cnt[1] = over;
          s_cnt[2] = over + c[e];
        }
      }
      meet();
      thr |= (uint32_t)s_cnt[0] << shift;
      above = s_cnt[1];
      reach = s_cnt[2];
      bit = shift - 1;
    }
  }
  int all = 0;
  auto before = [&](int mine) {  // sum of the threads' `mine` before this one; `all`: of all of them
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    all = __shfl_sync(0xffffffffu, upto, 31);
    int base = 0;
    if (W > 1) {
      if (lane == 0) s_pre[warp] = all;
      meet();
      const int x = lane < W ? s_pre[lane] : 0;
      base = __reduce_add_sync(0xffffffffu, lane < warp ? x : 0);
      all = __reduce_add_sync(0xffffffffu, x);
    }
    return base + upto - mine;
  };
  if (reach <= kShort && reach > 0) {  // gather the keys that reach the threshold, in index order
    from = max(from, thr);
    int mine = 0;
#pragma unroll
    for (int k = 0; k < KPT; ++k) mine += key[k] >= from;
    int at = before(mine);
#pragma unroll
    for (int k = 0; k < KPT; ++k)
      if (key[k] >= from) {
        s_key[at] = key[k];
        s_idx[at++] = j0 + k;
      }
    meet();
    if (warp != 0) return;
    constexpr int N = kShort / 32;
    uint32_t kk[N];
#pragma unroll
    for (int k = 0; k < N; ++k) kk[k] = k * 32 + lane < reach ? s_key[k * 32 + lane] : 0u;
    if (reach > A.top) {  // from the highest bit on which these differ, two bits at a time: three counts in one sum
      uint32_t o = 0, n = 0xffffffffu;
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (kk[k] != 0u && kk[k] != 0xffffffffu) o |= kk[k], n &= kk[k];
      o = __reduce_or_sync(0xffffffffu, o);
      n = __reduce_and_sync(0xffffffffu, n);
      bit = (o & ~n) ? 31 - __clz(o & ~n) : -1;
      thr = bit < 0 ? n : n & ~((2u << bit) - 1u);
      while (bit >= 0 && reach > A.top) {
        const int sh = max(bit - 1, 0);
        const uint32_t c1 = thr | (1u << sh), c2 = bit ? thr | (2u << sh) : c1, c3 = bit ? thr | (3u << sh) : c1;
        unsigned c = 0;  // at most kShort each: a byte holds it
#pragma unroll
        for (int k = 0; k < N; ++k)
          c += (kk[k] >= c1 ? 1u : 0u) + (kk[k] >= c2 ? 0x100u : 0u) + (kk[k] >= c3 ? 0x10000u : 0u);
        c = __reduce_add_sync(0xffffffffu, c);
        const int n1 = c & 255, n2 = (c >> 8) & 255, n3 = c >> 16;
        if (n3 >= A.top) thr = c3, reach = n3;
        else if (n2 >= A.top) thr = c2, reach = n2;
        else if (n1 >= A.top) thr = c1, reach = n1;
        bit = sh - 1;
      }
    } else {
      thr = 1;  // all of them, and nothing of the lanes without a key (0)
    }
    // reach > top now means equal keys at the threshold: the lowest indexes of them
    int gt_all = 0;
#pragma unroll
    for (int k = 0; k < N; ++k) gt_all += __popc(__ballot_sync(0xffffffffu, kk[k] > thr));
    const int need = reach > A.top ? A.top - gt_all : kShort;
    int gt_run = 0, eq_run = 0;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const bool gt = kk[k] > thr, eq = kk[k] == thr;
      const unsigned bg = __ballot_sync(0xffffffffu, gt), be = __ballot_sync(0xffffffffu, eq);
      const unsigned below = (1u << lane) - 1u;
      const int e0 = eq_run + __popc(be & below);
      if (gt || (eq && e0 < need)) {
        const int at = gt_run + __popc(bg & below) + min(e0, need), j = s_idx[k * 32 + lane];
        out[at] = j;
        if (out_s) out_s[at] = score[j];
      }
      gt_run += __popc(bg);
      eq_run += __popc(be);
    }
    return;
  }
  // the rest from the registers: keys above the threshold (low half) and equal to it (high)
  int mine = 0;
#pragma unroll
  for (int k = 0; k < KPT; ++k) mine += key[k] > thr ? 1 : key[k] == thr ? 1 << 16 : 0;
  const int first = before(mine);
  const int need = A.top - (all & 0xffff);  // equal keys to take
  int gt = first & 0xffff, eq = first >> 16;
#pragma unroll
  for (int k = 0; k < KPT; ++k) {
    const bool above = key[k] > thr, tie = key[k] == thr;
    if (above || (tie && eq < need)) {
      const int at = gt + min(eq, need), j = j0 + k;
      out[at] = j;
      if (out_s) out_s[at] = score[j];
    }
    gt += above;
    eq += tie;
  }
}

template <int KPT, Warps NW>
__global__ void __launch_bounds__(NW == Warps::MANY ? 1024 : 128) block_topk_regs_kernel(SelectArgs A, int W) {
  constexpr int ROWS = NW == Warps::ONE ? 4 : 1;  // rows per CTA
  __shared__ TopkShared<NW> sh[ROWS];
  ptx::grid_dependency_wait();
  const int64_t T = launch_length(A.T, A.len_dev, A.q_len);
  if (T == 0) {
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) set_length_error();
    return;
  }
  const int warp = threadIdx.x >> 5, r = NW == Warps::ONE ? warp : 0, i = (int)blockIdx.x * ROWS + r;
  if (i >= A.q_len) return;
  topk_row<KPT, NW>(A, T, blockIdx.y, i, A.score + ((int64_t)blockIdx.y * A.q_len + i) * A.ns, W,
                    NW == Warps::ONE ? 0 : warp, sh[r]);
}

// Scores and lists of one unit by one CTA, for a decode step's few query tokens
// (one row tile) and up to kOneBlocks blocks: the scores stay in shared memory,
// one launch and no workspace.  Bound by latency (a launch, the codes' loads, the
// search's meetings): one sequence of 8192 tokens 4.8 us, 16 of 32768 tokens 7.4
// us; as two kernels 2.6 us more each.
constexpr int kOneWarps = 16, kOneBlocks = 2048;

template <int KS, int GP>
__global__ void __launch_bounds__(kOneWarps * 32) block_select_one_kernel(SelectArgs A) {
  constexpr int STR = 2 * KS * 32 + 64;
  extern __shared__ __align__(16) unsigned char s_a[];  // int8 [16][STR], fp32 [16], fp32 scores [q_len][ns]
  __shared__ TopkShared<Warps::MANY> sh;
  float *s_sg = (float *)(s_a + 16 * STR), *s_score = s_sg + 16;
  const unsigned unit = blockIdx.x;
  ptx::grid_dependency_wait();
  const int64_t T = launch_length(A.T, A.len_dev, A.q_len);
  if (T == 0) {
    if (blockIdx.x == 0 && threadIdx.x == 0) set_length_error();
    return;
  }
  quantise_rows<KS, GP, kOneWarps>(A, unit, 0, 16, s_a, s_sg);
  __syncthreads();
  const int warp = threadIdx.x >> 5, j_end = (int)((unsigned)(T - 1) / (unsigned)A.bt) + 1;
  for (int j0 = warp * kScoreCols; j0 < j_end; j0 += kOneWarps * kScoreCols) {
    const BlockCodes<KS> f(A, unit, j0);
    score_tile<KS, GP>(A, f, s_a, s_sg, 0, j0, s_score + j0);
  }
  __syncthreads();
  const int W = (j_end + 127) / 128;  // four keys a thread
  if (warp >= W) return;
  for (int i = 0; i < A.q_len; ++i) {
    if (i) ptx::named_barrier_sync(1, W * 32);
    topk_row<4, Warps::MANY>(A, T, unit, i, s_score + i * A.ns, W, warp, sh);
  }
}

// The same for rows too long for registers: one CTA per row.  A radix select
// finds the key of the last one taken (4 passes of 8 bits), and an
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
  const float *score = A.score + row * A.ns;
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
// attention over the listed blocks: the general kernel (every layout).  Scalar
// lanes, one CTA per query head and part of the list, so K and V are decoded once
// per query head: one query of 4 kv-heads in groups of 16 over 32 blocks of 64
// takes 224 us, 16 queries of 8 heads of 64 over 64 blocks 2.7 ms
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

static bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

static int bounds_checks(const cq_paged_cache *cache, int64_t T, int32_t bt, const void *codes, const void *scales,
                         int64_t max_blocks, const char *what) {
  int r = validate_cache(cache);
  if (r) return r;
  const std::string w(what);
  CQ_REQUIRE(codes && scales, CQ_ERR_INVALID, w + ": null pointer");
  CQ_REQUIRE(aligned16(codes), CQ_ERR_INVALID, w + ": codes must be 16-byte aligned");
  CQ_REQUIRE(bt >= 1, CQ_ERR_INVALID, w + ": block_tokens must be >= 1");
  CQ_REQUIRE(T >= 1 && T <= (int64_t)cache->max_pages * cache->page_tokens, CQ_ERR_INVALID,
             w + ": tokens beyond the mapped pages (or none)");
  CQ_REQUIRE((T - 1) / bt < max_blocks, CQ_ERR_INVALID, w + ": max_blocks too small");
  CQ_REQUIRE((T - 1) / bt < (1LL << 30), CQ_ERR_UNSUPPORTED, w + ": too many blocks");
  return CQ_OK;
}

static int launch_bounds(const sparse::BoundsArgs &A, cudaStream_t st, const char *what) {
  const int64_t units = (int64_t)A.cv.B * A.cv.H;
  CQ_REQUIRE(units < (1LL << 31), CQ_ERR_INVALID, std::string(what) + ": grid too large");
  const int64_t grid = units * A.nb;
  CQ_REQUIRE(grid < (1LL << 31), CQ_ERR_INVALID, std::string(what) + ": grid too large");
  const CompView &c = A.cv.c[0];
  const int D = A.cv.D, rows = D == 64 ? 4 : D == 128 ? 2 : 1;  // code rows a warp takes at once
  if ((D == 64 || D == 128 || D == 256) && c.order == CQ_ORDER_NATURAL && c.stok && c.stride % rows == 0 &&
      c.stride > 1 && A.bt % rows == 0 && aligned16(c.kf) && (c.kf_hs | c.kf_cs) % 8 == 0 &&
      A.T + A.bt < (1LL << 31) && units <= 65535) {
    auto *fn = D == 64    ? sparse::block_bounds_rows_kernel<64>
               : D == 128 ? sparse::block_bounds_rows_kernel<128>
                          : sparse::block_bounds_rows_kernel<256>;
    return launch_after(fn, dim3((unsigned)((A.nb - 1) / 4 + 1), (unsigned)units), 128, 0, st, what, A);
  }
  const int threads = (A.cv.D + 31) & ~31;
  return launch_after(sparse::block_bounds_kernel, dim3((unsigned)grid), threads, 0, st, what, A);
}

extern "C" int cq_block_bounds(const cq_paged_cache *cache, int64_t t0, int64_t T, int32_t block_tokens, int8_t *codes,
                               float *scales, int64_t max_blocks, void *stream) {
  int r = bounds_checks(cache, T, block_tokens, codes, scales, max_blocks, "cq_block_bounds");
  if (r) return r;
  CQ_REQUIRE(t0 >= 0 && t0 <= T, CQ_ERR_INVALID, "cq_block_bounds: t0 must lie in [0, T]");
  if (t0 == T) return CQ_OK;
  sparse::BoundsArgs A{make_view(*cache), t0,   T,     nullptr, 0, block_tokens, 0, t0 / block_tokens,
                       codes,             scales, max_blocks};
  A.nb = (int)((T - 1) / block_tokens - t0 / block_tokens + 1);
  return launch_bounds(A, (cudaStream_t)stream, "cq_block_bounds");
}

extern "C" int cq_block_bounds_at(const cq_paged_cache *cache, const int64_t *len_dev, int64_t max_len, int32_t S,
                                  int32_t block_tokens, int8_t *codes, float *scales, int64_t max_blocks,
                                  void *stream) {
  int r = bounds_checks(cache, max_len, block_tokens, codes, scales, max_blocks, "cq_block_bounds_at");
  if (r) return r;
  CQ_REQUIRE(len_dev && S >= 1 && S <= max_len, CQ_ERR_INVALID, "cq_block_bounds_at: bad length arguments");
  sparse::BoundsArgs A{make_view(*cache), 0,    max_len, len_dev, S, block_tokens, 0, 0,
                       codes,             scales, max_blocks};
  A.nb = (int)(((int64_t)S + block_tokens - 2) / block_tokens + 1);  // the most blocks S tokens can touch
  return launch_bounds(A, (cudaStream_t)stream, "cq_block_bounds_at");
}

extern "C" int cq_block_bounds_read(const int8_t *codes, const float *scales, int64_t units, int64_t max_blocks,
                                    int64_t first, int64_t n, int32_t head_dim, float *out, void *stream) {
  CQ_REQUIRE(codes && scales && out, CQ_ERR_INVALID, "cq_block_bounds_read: null pointer");
  CQ_REQUIRE(aligned16(codes) && aligned16(out), CQ_ERR_INVALID,
             "cq_block_bounds_read: codes and out must be 16-byte aligned");
  CQ_REQUIRE(units >= 1 && first >= 0 && n >= 0 && n <= max_blocks - first && head_dim >= 8 && head_dim <= 256,
             CQ_ERR_INVALID, "cq_block_bounds_read: bad sizes");
  if (n == 0) return CQ_OK;
  CQ_REQUIRE(n <= (1LL << 33) / units, CQ_ERR_INVALID, "cq_block_bounds_read: grid too large");
  const int64_t grid = (units * n + 7) / 8;  // a warp per block
  return launch_after(sparse::bounds_read_kernel, dim3((unsigned)grid), 256, 0, (cudaStream_t)stream,
                      "cq_block_bounds_read", codes, scales, units, max_blocks, first, n, head_dim, out);
}

// The form of a selection: the head groups' power of two (its log), whether the tensor-core kernels take it, whether
// one CTA per unit does it all.
struct SelectForm {
  int lg = 0;
  bool mma = false, one = false;
  int64_t n = 0, ns = 0;
  size_t bytes = 0;  // workspace
};

static int select_form(int32_t batch, int32_t kv_heads, int32_t head_dim, int32_t n_q_heads, int32_t q_len, int64_t T,
                       int32_t block_tokens, SelectForm &f) {
  CQ_REQUIRE(batch >= 1 && kv_heads >= 1 && block_tokens >= 1, CQ_ERR_INVALID, "cq_block_select: bad sizes");
  CQ_REQUIRE(head_dim >= 8 && head_dim <= 256 && head_dim % 8 == 0, CQ_ERR_UNSUPPORTED,
             "cq_block_select: head_dim must be a multiple of 8 in [8, 256]");
  CQ_REQUIRE(n_q_heads >= 1 && n_q_heads % kv_heads == 0, CQ_ERR_INVALID,
             "cq_block_select: n_q_heads must be a positive multiple of kv_heads");
  CQ_REQUIRE(q_len >= 1 && q_len <= T, CQ_ERR_INVALID, "cq_block_select: need 1 <= q_len <= T");
  f.n = (T - 1) / block_tokens + 1;
  CQ_REQUIRE(f.n < (1LL << 30), CQ_ERR_INVALID, "cq_block_select: too many blocks");
  f.ns = (f.n + 7) & ~7LL;
  const int G = n_q_heads / kv_heads;
  while ((1LL << f.lg) < G) ++f.lg;
  const int64_t units = (int64_t)batch * kv_heads;
  CQ_REQUIRE(units < (1LL << 31) && units * q_len < (1LL << 31), CQ_ERR_UNSUPPORTED,
             "cq_block_select: too many query tokens");
  f.mma = (head_dim == 64 || head_dim == 96 || head_dim == 128 || head_dim == 256) && G <= 16 && units < 65536 &&
          T < (1LL << 31);
  // one CTA scores up to 256 blocks a pass; longer rows want the whole machine unless there are units for it
  f.one = f.mma && ((int64_t)q_len << f.lg) <= 16 && f.n <= sparse::kOneBlocks && q_len * f.ns <= 8192 &&
          (f.n <= 512 || 2 * units >= sm_count());
  f.bytes = f.one ? 0 : (size_t)units * q_len * f.ns * sizeof(float);
  return CQ_OK;
}

extern "C" int cq_block_select_workspace(int32_t batch, int32_t kv_heads, int32_t head_dim, int32_t n_q_heads,
                                         int32_t q_len, int64_t T, int32_t block_tokens, size_t *bytes) {
  CQ_REQUIRE(bytes, CQ_ERR_INVALID, "cq_block_select_workspace: bytes is null");
  SelectForm f;
  int r = select_form(batch, kv_heads, head_dim, n_q_heads, q_len, T, block_tokens, f);
  if (r) return r;
  *bytes = f.bytes;
  return CQ_OK;
}

// One entry per head size (64, 96, 128, 256) and power of two of the group.
static int size_index(int D) { return D == 64 ? 0 : D == 96 ? 1 : D == 128 ? 2 : 3; }
#define CQ_BY_GROUP(K, KS) {K<KS, 1>, K<KS, 2>, K<KS, 4>, K<KS, 8>, K<KS, 16>}
#define CQ_BY_SIZE(K) {CQ_BY_GROUP(K, 2), CQ_BY_GROUP(K, 3), CQ_BY_GROUP(K, 4), CQ_BY_GROUP(K, 8)}

static int launch_one(const sparse::SelectArgs &A, const SelectForm &f, cudaStream_t st) {
  using namespace sparse;
  using Fn = void (*)(SelectArgs);
  static const Fn table[4][5] = CQ_BY_SIZE(block_select_one_kernel);
  const size_t smem = 16 * (2 * A.D + 64 + 4) + (size_t)A.q_len * A.ns * sizeof(float);  // below 43 KB
  return launch_after(table[size_index(A.D)][f.lg], dim3((unsigned)(A.B * A.H)), kOneWarps * 32, smem, st,
                      "cq_block_select", A);
}

static int launch_scores(const sparse::SelectArgs &A, const SelectForm &f, cudaStream_t st) {
  using namespace sparse;
  const int64_t rows = (int64_t)A.B * A.H * A.q_len, units = (int64_t)A.B * A.H;
  if (f.mma) {
    using Fn = void (*)(SelectArgs, int, int);
    static const Fn table[4][5] = CQ_BY_SIZE(block_score_mma_kernel);
    const int tpt = 16 >> f.lg, row_tiles = (A.q_len - 1) / tpt + 1;
    // A CTA's rows are quantised once for all its columns, so it takes many columns as soon as there are two
    // CTAs per SM without splitting them; few row tiles, so that this happens early
    const int tiles = std::min(row_tiles, 4);
    const int64_t groups = ((int64_t)row_tiles + tiles - 1) / tiles;
    CQ_REQUIRE(groups < 65536, CQ_ERR_UNSUPPORTED, "cq_block_select: too many query tokens");
    const int per = kScoreWarps * kScoreCols;
    const int64_t cols = (A.n + per - 1) / per;
    const int64_t split = std::max<int64_t>(1, std::min<int64_t>(cols, 2 * sm_count() / (groups * units)));
    const int passes = (int)((cols + split - 1) / split);
    const dim3 grid((unsigned)((cols + passes - 1) / passes), (unsigned)groups, (unsigned)units);
    return launch_after(table[size_index(A.D)][f.lg], grid, kScoreWarps * 32,
                        (size_t)tiles * 16 * (2 * A.D + 64 + 4), st, "cq_block_select", A, tiles, passes);
  }
  const int64_t grid = (rows * A.n + 7) / 8;
  CQ_REQUIRE(grid < (1LL << 31), CQ_ERR_UNSUPPORTED, "cq_block_select: too many scores");
  block_score_kernel<<<(unsigned)grid, 256, 0, st>>>(A);
  return check_launch("cq_block_select");
}

static int launch_topk(const sparse::SelectArgs &A, int64_t rows, cudaStream_t st) {
  using namespace sparse;
  const int64_t units = (int64_t)A.B * A.H;
  if (A.n > 16 * 1024 || A.T >= (1LL << 31) || units > 65535) {
    block_topk_kernel<<<(unsigned)rows, 256, 0, st>>>(A);
    return check_launch("cq_block_select");
  }
  // a warp a row from 12 rows per SM on (1024 blocks: 1184 rows 6.7 us against 6.2 with four warps, 2400 rows 9.3
  // against 10.0; up to 256 blocks the same either way)
  if (A.n > 256 && A.n <= 1024 && rows >= 12 * sm_count()) {
    auto *fn = A.n <= 512 ? block_topk_regs_kernel<16, Warps::ONE> : block_topk_regs_kernel<32, Warps::ONE>;
    return launch_after(fn, dim3(((unsigned)A.q_len + 3) / 4, (unsigned)units), 128, 0, st, "cq_block_select", A, 1);
  }
  // keys a thread: four, or where rows abound so many that up to four warps hold a row (320 rows of 2048 blocks 5.2
  // us against 6.2, 4096 rows 19.4 against 24)
  int kpt = 4;
  if (A.n > 128 && A.n <= 4096 && rows >= 2 * sm_count()) kpt = A.n <= 1024 ? 8 : A.n <= 2048 ? 16 : 32;
  while (A.n > (int64_t)kpt * 32 * 32) kpt *= 2;  // up to 16
  const int W = (int)((A.n + kpt * 32 - 1) / (kpt * 32));
  using Fn = void (*)(SelectArgs, int);
  static const Fn few[4] = {block_topk_regs_kernel<4, Warps::FEW>, block_topk_regs_kernel<8, Warps::FEW>,
                            block_topk_regs_kernel<16, Warps::FEW>, block_topk_regs_kernel<32, Warps::FEW>};
  static const Fn many[3] = {block_topk_regs_kernel<4, Warps::MANY>, block_topk_regs_kernel<8, Warps::MANY>,
                             block_topk_regs_kernel<16, Warps::MANY>};
  const int size = kpt == 4 ? 0 : kpt == 8 ? 1 : kpt == 16 ? 2 : 3;
  return launch_after(W <= 4 ? few[size] : many[size], dim3((unsigned)A.q_len, (unsigned)units), W * 32, 0, st,
                      "cq_block_select", A, W);
}

extern "C" int cq_block_select(const int8_t *codes, const float *scales, int64_t max_blocks, int32_t block_tokens,
                               int32_t batch, int32_t kv_heads, int32_t head_dim, int64_t T, const int64_t *len_dev,
                               const void *q, int q_dtype, int32_t n_q_heads, int32_t q_len, int64_t q_sb,
                               int64_t q_sh, int64_t q_sq, const int64_t *starts, int32_t first, int32_t recent,
                               int32_t top, int32_t *blocks, float *block_scores, void *workspace,
                               size_t workspace_bytes, void *stream) {
  SelectForm f;
  int r = select_form(batch, kv_heads, head_dim, n_q_heads, q_len, T, block_tokens, f);
  if (r) return r;
  CQ_REQUIRE(codes && scales && q && blocks, CQ_ERR_INVALID, "cq_block_select: null pointer");
  CQ_REQUIRE(aligned16(codes), CQ_ERR_INVALID, "cq_block_select: codes must be 16-byte aligned");
  CQ_REQUIRE(q_dtype == CQ_F16 || q_dtype == CQ_BF16, CQ_ERR_UNSUPPORTED, "cq_block_select: q dtype must be f16/bf16");
  CQ_REQUIRE(first >= 0 && recent >= 0 && top >= 1 && first <= top && recent <= top - first, CQ_ERR_INVALID,
             "cq_block_select: need first + recent <= top");
  CQ_REQUIRE(top <= sparse::kMaxTop, CQ_ERR_UNSUPPORTED, "cq_block_select: top must be <= 4096");
  CQ_REQUIRE(f.n <= max_blocks, CQ_ERR_INVALID, "cq_block_select: T beyond the summarised blocks");
  CQ_REQUIRE(f.bytes == 0 || (workspace && workspace_bytes >= f.bytes), CQ_ERR_WORKSPACE,
             "cq_block_select: workspace too small");
  CQ_REQUIRE(f.bytes == 0 || aligned16(workspace), CQ_ERR_INVALID, "cq_block_select: workspace must be 16-byte aligned");
  sparse::SelectArgs A{codes,  scales, max_blocks, block_tokens, batch, kv_heads, head_dim, n_q_heads / kv_heads,
                       q_len,  T,      len_dev,    q,            q_dtype, q_sb,   q_sh,     q_sq,
                       starts, first,  recent,     top,          blocks,  block_scores,     f.n, f.ns, (float *)workspace};
  cudaStream_t st = (cudaStream_t)stream;
  if (f.one) return launch_one(A, f, st);
  r = launch_scores(A, f, st);
  if (r) return r;
  return launch_topk(A, (int64_t)batch * kv_heads * q_len, st);
}

static int sparse_checks(const cq_paged_cache *cache, int64_t T, int32_t n_q_heads, int32_t q_len, int32_t top,
                         int32_t bt) {
  int r = validate_cache(cache);
  if (r) return r;
  CQ_REQUIRE(n_q_heads >= 1 && n_q_heads % cache->kv_heads == 0, CQ_ERR_INVALID,
             "cq_sparse_attention: n_q_heads must be a positive multiple of kv_heads");
  CQ_REQUIRE(q_len >= 1 && q_len <= T, CQ_ERR_INVALID, "cq_sparse_attention: need 1 <= q_len <= T");
  CQ_REQUIRE(T <= (int64_t)cache->max_pages * cache->page_tokens, CQ_ERR_INVALID,
             "cq_sparse_attention: T beyond mapped pages");
  const int64_t heads = (int64_t)cache->batch * n_q_heads;
  CQ_REQUIRE(heads < (1LL << 31) && heads * q_len < (1LL << 31), CQ_ERR_UNSUPPORTED,
             "cq_sparse_attention: too many query tokens");
  CQ_REQUIRE(top >= 1 && bt >= 1, CQ_ERR_INVALID, "cq_sparse_attention: bad list length or block_tokens");
  CQ_REQUIRE(top <= sparse::kMaxTop, CQ_ERR_UNSUPPORTED, "cq_sparse_attention: at most 4096 blocks per list");
  return CQ_OK;
}

extern "C" int cq_sparse_attention_workspace(const cq_paged_cache *cache, int64_t T, int32_t n_q_heads, int32_t q_len,
                                             int32_t top, int32_t block_tokens, size_t *bytes) {
  int r = sparse_checks(cache, T, n_q_heads, q_len, top, block_tokens);
  if (r) return r;
  CQ_REQUIRE(bytes, CQ_ERR_INVALID, "cq_sparse_attention_workspace: bytes is null");
  if (sparse_fast_supported(*cache, T, n_q_heads, block_tokens)) {
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
  if (sparse_fast_supported(*cache, T, n_q_heads, block_tokens))
    return run_sparse_fast(*cache, T, len_dev, q, q_dtype, n_q_heads, q_len, q_sb, q_sh, q_sq, scale, starts, blocks,
                           top, block_tokens, out, out_dtype, lse_out, (cudaStream_t)stream);
  const int splits = sparse::pick_list_splits(rows, top), D = cache->head_dim;
  CQ_REQUIRE(workspace && workspace_bytes >= sparse::generic_bytes(rows, splits, D), CQ_ERR_WORKSPACE,
             "cq_sparse_attention: workspace too small");
  CQ_REQUIRE(((uintptr_t)workspace & 3) == 0, CQ_ERR_INVALID, "cq_sparse_attention: workspace must be 4-byte aligned");
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
