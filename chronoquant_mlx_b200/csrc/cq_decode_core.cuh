// cq_decode_core.cuh -- the warp-level core of attention over chunk blocks of
// the compressed cache: the chunk geometry, the scores and softmax of 32
// tokens, the output of 16 tokens and the per-warp partial.  The dense decode
// kernel (cq_decode_fast.cu, which explains the method) and the block-sparse
// one (cq_sparse_fast.cu) are built from it.
#pragma once

#include "cq_common.cuh"
#include "cq_ptx.cuh"

namespace cq {
namespace fast {

constexpr int HD = 128;          // head_dim
constexpr int kMaxWarps = 16;    // warps per CTA (one CTA per SM)
constexpr float TAU = 8.0f;      // lazy-rescale threshold (log2 units)
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr long long WAIT_BUDGET = 1LL << 31;  // clock cycles (~1 s) before a wait gives up
constexpr int ERR_TIMEOUT_FULL = 1;
constexpr int ERR_LENGTH = 4;  // a device-resident length outside [1, mapped tokens]
constexpr int kQaBytes = 16 * 8 * 4;  // per-warp q.anchor table: 16 anchors x 8 heads, fp32
constexpr int kQnBytes = 8 * 32 * 8;  // per-warp natural-order query fragments
constexpr int kBarsPerWarp = 4;       // a warp's copy barriers (at most two slots, or one K and one V buffer)

constexpr int cx_log2(int x) { return x <= 1 ? 0 : 1 + cx_log2(x >> 1); }
constexpr int cx_up16(int x) { return (x + 15) & ~15; }
constexpr int cx_max(int a, int b) { return a > b ? a : b; }

// Compile-time geometry of one (stride_k, stride_v) pair: chunk tokens, tiles
// per chunk, anchors per chunk and the byte offsets of a chunk block's six
// segments [K anchors][K codes][K scales][V anchors][V codes][V scales]
// (each 16-byte aligned) -- the layout the cache stores and a slot mirrors.
template <int SK_, int SV_, int VP_ = 4>
struct Geo {
  static constexpr int SK = SK_, SV = SV_;
  // VP: bits per stored V code -- 4 (INT4 lanes, 64-byte rows), or bit planes of physical 3-bit
  // (CQ_ORDER_PLANES3, 48 bytes) or 2-bit codes (CQ_ORDER_PLANES2, 32 bytes)
  static constexpr int VP = VP_;
  static constexpr bool V3 = VP == 3, PL = VP < 4;
  static constexpr int VR = VP == 3 ? 48 : VP == 2 ? 32 : HD / 2;
  static constexpr int LSK = cx_log2(SK), LSV = cx_log2(SV);
  static constexpr int C = cx_max(32, cx_max(SK, SV));
  static constexpr int NT = C / 16;
  static constexpr int AK = C / SK, AV = C / SV;
  static constexpr int O_KF0 = 0;
  static constexpr int O_CD0 = cx_up16(O_KF0 + AK * HD * 2);
  static constexpr int O_SC0 = cx_up16(O_CD0 + (C - AK) * (HD / 2));
  static constexpr int O_KF1 = cx_up16(O_SC0 + C * 2);
  static constexpr int O_CD1 = cx_up16(O_KF1 + AV * HD * 2);
  static constexpr int O_SC1 = cx_up16(O_CD1 + (C - AV) * VR);
  static constexpr int SLOT = cx_up16(O_SC1 + C * 2);
  // 32-token chunks: two slots per warp, each filled with a whole block.
  // 64-token chunks (SPLIT): the K part [0, O_KF1) and the V part [O_KF1,
  // SLOT) of a block go to separate buffers, one of each per warp; the K
  // buffer is refilled as soon as the chunk's scores are done and the V
  // buffer once its output is accumulated, so a warp needs one block of
  // buffers instead of two and 16 warps fit in shared memory.
  static constexpr bool SPLIT = C == 64;
  static constexpr int KB = O_KF1, VB = SLOT - O_KF1;
  static constexpr int V_CD = O_CD1 - O_KF1, V_SC = O_SC1 - O_KF1;  // offsets inside the V part
  static constexpr int NSK = SPLIT ? 1 : 2;                         // buffer pairs (SPLIT) or slots
  static constexpr int BUF = NSK * SLOT;                            // a warp's copy buffers
  static_assert(SK >= 16 && SV >= 8 && C <= 64 && AK <= 16, "geometry outside the kernel's range");
  static_assert(KB % 16 == 0 && VB % 16 == 0, "bulk copies need 16-byte sizes");
};

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct QFrag {
  uint32_t qb[4][4];  // query as B fragments in the K-code order (q/16 on the 16n lanes)
  float2 qc;          // q . (raw values of the all-8 word) for heads 2t, 2t+1
};

// One query token of a GQA group: head g, dim d at q[base + g * sh + d].
struct QuerySrc {
  const void *q;
  int64_t base, sh;
  int dtype, gqa;
  float scale;
};

__device__ __forceinline__ float q_scaled(const QuerySrc &s, int g, int d) {
  const float sc = round_dt(s.scale, s.dtype);
  float v = load_as_float(s.q, s.base + g * s.sh + d, s.dtype) * sc;
  return round_dt(v, s.dtype);  // q * scale in the query dtype (attention.py:46)
}

// Loads a unit's query: K-code-order fragments into registers, natural-order
// fragments (for the anchors) into the warp's table qn[8][32 lanes] (uint2).
__device__ __forceinline__ void load_q(const QuerySrc &p, int lane, QFrag &f, uint2 *qn) {
  const int g = lane >> 2, t = lane & 3;
  const bool real = g < p.gqa;
  float cc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int J = 0; J < 4; ++J) {
    const int d0 = 32 * t + 8 * J;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = real ? q_scaled(p, g, d0 + i) : 0.f;
    f.qb[J][0] = ptx::pack_half2(v[0], v[4]);
    f.qb[J][1] = ptx::pack_half2(v[1] * 0.0625f, v[5] * 0.0625f);
    f.qb[J][2] = ptx::pack_half2(v[2], v[6]);
    f.qb[J][3] = ptx::pack_half2(v[3] * 0.0625f, v[7] * 0.0625f);
    ptx::mma_f16_16816(cc, ptx::RAW_CODE0_LO, ptx::RAW_CODE0_LO, ptx::RAW_CODE0_HI, ptx::RAW_CODE0_HI, f.qb[J][0],
                       f.qb[J][1]);
    ptx::mma_f16_16816(cc, ptx::RAW_CODE0_LO, ptx::RAW_CODE0_LO, ptx::RAW_CODE0_HI, ptx::RAW_CODE0_HI, f.qb[J][2],
                       f.qb[J][3]);
  }
  f.qc = make_float2(cc[0], cc[1]);
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) {
    const int d0 = 16 * kk + 2 * t;
    qn[kk * 32 + lane] =
        real ? make_uint2(ptx::pack_half2(q_scaled(p, g, d0), q_scaled(p, g, d0 + 1)),
                          ptx::pack_half2(q_scaled(p, g, d0 + 8), q_scaled(p, g, d0 + 9)))
             : make_uint2(0u, 0u);
  }
}

// q . anchor (log2 units) for the first nK (<= 16) K anchors of a slot, as
// one MMA tile with rows = anchors; table [16][8] fp32 at `qa`.
// frag(kk): the query's B fragment of channels 16 kk .. 16 kk + 15.
template <class Frag>
__device__ __forceinline__ void compute_qa_from(uint32_t kfK, float *qa, int nK, Frag frag, int lane) {
  const int g = lane >> 2, t = lane & 3;
  const int mi = lane >> 3, rr = lane & 7;
  float c0[4] = {0.f, 0.f, 0.f, 0.f}, c1[4] = {0.f, 0.f, 0.f, 0.f};
  const int arow = min(rr + ((mi & 1) ? 8 : 0), nK - 1);
  const uint32_t base = kfK + arow * (HD * 2) + ((mi & 2) ? 16 : 0);
#pragma unroll
  for (int kk = 0; kk < 8; kk += 2) {
    uint32_t a0, a1, a2, a3, b0, b1, b2, b3;
    ptx::ldmatrix_x4(a0, a1, a2, a3, base + kk * 32);
    ptx::ldmatrix_x4(b0, b1, b2, b3, base + kk * 32 + 32);
    const uint2 q0 = frag(kk), q1 = frag(kk + 1);
    ptx::mma_f16_16816(c0, a0, a1, a2, a3, q0.x, q0.y);
    ptx::mma_f16_16816(c1, b0, b1, b2, b3, q1.x, q1.y);
  }
  float *row0 = qa + g * 8 + 2 * t;
  *(float2 *)row0 = make_float2((c0[0] + c1[0]) * LOG2E, (c0[1] + c1[1]) * LOG2E);
  *(float2 *)(row0 + 64) = make_float2((c0[2] + c1[2]) * LOG2E, (c0[3] + c1[3]) * LOG2E);
}

__device__ __forceinline__ void compute_qa(uint32_t kfK, float *qa, int nK, const uint2 *qn, int lane) {
  compute_qa_from(kfK, qa, nK, [&](int kk) { return qn[kk * 32 + lane]; }, lane);
}

// A query kept as a tile in shared memory instead: fp16 [8 heads][kQRow bytes],
// rows 16 bytes apart modulo 128, from which fragments are read without bank
// conflicts.  It is filled with 8-byte loads where the rows allow them.
constexpr int kQRow = HD * 2 + 16, kQTileBytes = 8 * kQRow;

__device__ __forceinline__ void load_q_tile(const QuerySrc &p, int lane, QFrag &f, unsigned char *tile) {
  const bool quads = (((uintptr_t)p.q & 7) | (p.base & 3) | (p.sh & 3)) == 0;
  const float sc = round_dt(p.scale, p.dtype);
  uint2 raw[8];
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    raw[g] = make_uint2(0u, 0u);
    if (g < p.gqa) {
      const uint16_t *src = (const uint16_t *)p.q + p.base + g * p.sh + 4 * lane;
      if (quads)
        raw[g] = *(const uint2 *)src;
      else
        raw[g] = make_uint2((uint32_t)src[0] | (uint32_t)src[1] << 16, (uint32_t)src[2] | (uint32_t)src[3] << 16);
    }
  }
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t u = (uint16_t)((i & 2 ? raw[g].y : raw[g].x) >> (i & 1 ? 16 : 0));
      const float x = p.dtype == CQ_BF16 ? __uint_as_float((uint32_t)u << 16) : __half2float(__ushort_as_half(u));
      v[i] = round_dt(x * sc, p.dtype);  // q * scale in the query dtype (attention.py:46)
    }
    *(uint2 *)(tile + g * kQRow + 8 * lane) = make_uint2(ptx::pack_half2(v[0], v[1]), ptx::pack_half2(v[2], v[3]));
  }
  __syncwarp();
  const int g = lane >> 2, t = lane & 3;
  float cc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int J = 0; J < 4; ++J) {  // the K-code order, as load_q<false>
    const uint4 w = *(const uint4 *)(tile + g * kQRow + 64 * t + 16 * J);
    f.qb[J][0] = __byte_perm(w.x, w.z, 0x5410u);
    f.qb[J][1] = __byte_perm(w.x, w.z, 0x7632u);
    f.qb[J][2] = __byte_perm(w.y, w.w, 0x5410u);
    f.qb[J][3] = __byte_perm(w.y, w.w, 0x7632u);
    constexpr uint32_t EIGHT = 0x00080008u;  // 8 * 2^-24, as the codes come
    ptx::mma_f16_16816(cc, EIGHT, EIGHT, EIGHT, EIGHT, f.qb[J][0], f.qb[J][1]);
    ptx::mma_f16_16816(cc, EIGHT, EIGHT, EIGHT, EIGHT, f.qb[J][2], f.qb[J][3]);
  }
  f.qc = make_float2(cc[0], cc[1]);
}

__device__ __forceinline__ void compute_qa_tile(uint32_t kfK, float *qa, int nK, const unsigned char *tile, int lane) {
  const unsigned char *at = tile + (lane >> 2) * kQRow + 4 * (lane & 3);
  compute_qa_from(
      kfK, qa, nK,
      [&](int kk) { return make_uint2(*(const uint32_t *)(at + 32 * kk), *(const uint32_t *)(at + 32 * kk + 16)); },
      lane);
}

// ---------------------------------------------------------------------------
// per-warp softmax state and one chunk of NT 16-token tiles
// ---------------------------------------------------------------------------
struct WarpState {
  float m[2];     // running max (log2 units) of heads 2t, 2t+1
  float l[2];     // this thread's partial sums
  float o[8][4];  // O^T fragments: [m-tile i][c0..c3]
  float vb[4];    // 72 * sum of the fp16 code weights P' (same fragment layout): the V code offset
  float ps[4];    // P summed per V anchor slot of the chunk (rows) and head
};

__device__ __forceinline__ void reset(WarpState &st) {
  st.m[0] = st.m[1] = -INFINITY;
  st.l[0] = st.l[1] = 0.f;
  st.vb[0] = st.vb[1] = st.vb[2] = st.vb[3] = 0.f;
  st.ps[0] = st.ps[1] = st.ps[2] = st.ps[3] = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) st.o[i][j] = 0.f;
}

// Per-lane shared-memory byte addresses into a K part.  Code rows are stored
// in P-frame order; the row of chunk-local token x is x - x/stride - 1 (an
// I-frame lands on the previous row, read harmlessly with scale 0).  For a
// 16-token tile at tb with stride_k >= 16 the K rows of tokens tb + x are
// (tb - tb/stride_k) + x - 1.
struct KAddr {
  uint32_t cdK;  // K code row of token g (tile base 0), word group t
  uint32_t scK;  // K scale of token g
  uint32_t qa;   // q.anchor table, heads 2t, 2t+1
  template <class G>
  __device__ __forceinline__ KAddr(G, uint32_t kb, uint32_t qa_base, int lane) {
    const int g = lane >> 2, t = lane & 3;
    cdK = kb + G::O_CD0 + (g - 1) * 64 + t * 16;
    scK = kb + G::O_SC0 + g * 2;
    qa = qa_base + t * 8;
  }
};

// Per-lane shared-memory byte addresses into a V part.
struct VAddr {
  uint32_t cdV;   // V code row of token 2t (tile base 0), words 2g, 2g+1
  uint32_t scV;   // V scales of tokens 2t, 2t+1 (one 32-bit word)
  uint32_t kfV;   // V anchor row of this lane's ldmatrix row (tile 0)
  uint32_t kfV0;  // V anchor row 0, same column half
  int dv8;        // V rows between tokens 2t and 2t+8
  template <class G>
  __device__ __forceinline__ VAddr(G, uint32_t vb, int lane) {
    const int g = lane >> 2, t = lane & 3, mi = lane >> 3;
    constexpr bool v8 = G::LSV == 3;
    cdV = vb + G::V_CD + (2 * t - 1) * G::VR + (G::PL ? 0 : g * 8);  // bit-plane rows: lane offsets at use
    dv8 = v8 ? 7 : 8;
    scV = vb + G::V_SC + t * 4;
    kfV0 = vb + ((mi & 1) ? 16 : 0);
    kfV = kfV0 + ((v8 ? (mi >> 1) : 0) * (HD * 2));
  }
};

__device__ __forceinline__ float lds_half_as_float(uint32_t a) {
  unsigned short v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a));
  return __half2float(__ushort_as_half(v));
}

// Scores of the two 16-token tiles at chunk-local token t0 and their softmax
// update; P of the two tiles in the MMA B-operand layout (a lane holds tokens
// 2t, 2t+1 (and 2t+8, 2t+9) of head g) into bp[0..1].  When the running max
// moves, the output state is rescaled and the function returns true with the
// factor for head g in `fh` (for the P of the chunk's earlier groups).
// MASK: 0 every token of the chunk counts, 1 tokens below nvalid, 2 tokens
// from vlo on and below nvalid (one of this group's at least).
// RAW: K codes enter the score MMAs as 1024 + n and 1024 + 16n (load_q's
// fragments; the sums reach 1032 sum|q|, whose fp32 rounding shows in the scores);
// otherwise as the nibbles alone (load_q_tile's fragments): the bits of n and 16n
// in a half are the subnormal numbers n * 2^-24 and 16n * 2^-24, exact operands
// without an offset, summed apart and weighted by 2^24 and 2^20 with the scale
// (sums of at most 15 sum|q|; as 64 + n, with sums of 79 sum|q|, 4096 units of 32
// chunks took 221 us, so 217).
template <class G, int MASK, bool RAW = true>
__device__ __forceinline__ bool k_group(WarpState &st, const KAddr &A, const QFrag &f, int t0, int nvalid, int lane,
                                        uint2 (&bp)[2], __half2 &fh, int vlo = 0) {
  constexpr int lsk = G::LSK;
  constexpr int NT = 2;
  const int g = lane >> 2;
  float s[NT][4];
  // ---------------- scores S^T[token][head] = scale_t * (q.codes_t) + q.anchor
#pragma unroll
  for (int tile = 0; tile < NT; ++tile) {
    const int tb = t0 + tile * 16;
    const uint32_t rk = (uint32_t)((tb - (tb >> lsk)) * 64);  // K rows before the tile
    const uint4 wk0 = ptx::lds_u128(A.cdK + rk);
    const uint4 wk1 = ptx::lds_u128(A.cdK + rk + 8 * 64);
    constexpr float UNIT = RAW ? LOG2E : LOG2E * 16777216.f;
    const float sk0 = lds_half_as_float(A.scK + tb * 2) * UNIT;
    const float sk1 = lds_half_as_float(A.scK + (tb + 8) * 2) * UNIT;
    const float2 qa = ptx::lds_f2(A.qa + (uint32_t)((tb >> lsk) * 32));  // one K anchor per tile (stride >= 16)
    // raw nibbles (1024+n, 1024+16n) against q (q/16 on the 16n lanes); the
    // accumulator starts at -q.(all-8 word), which removes the raw offset
    float ca[4] = {-f.qc.x, -f.qc.y, -f.qc.x, -f.qc.y}, cb[4] = {0.f, 0.f, 0.f, 0.f};
    const uint32_t w0[4] = {wk0.x, wk0.y, wk0.z, wk0.w};
    const uint32_t w1[4] = {wk1.x, wk1.y, wk1.z, wk1.w};
#pragma unroll
    for (int J = 0; J < 4; ++J) {
      if constexpr (RAW) {
        uint32_t h0[4], h1[4];
        ptx::nibbles_to_half2_raw(w0[J], h0);  // (d0,d4) (d1,d5) (d2,d6) (d3,d7)
        ptx::nibbles_to_half2_raw(w1[J], h1);
        ptx::mma_f16_16816(ca, h0[0], h1[0], h0[1], h1[1], f.qb[J][0], f.qb[J][1]);
        ptx::mma_f16_16816(cb, h0[2], h1[2], h0[3], h1[3], f.qb[J][2], f.qb[J][3]);
      } else {
        constexpr uint32_t EVEN = 0x000f000fu, ODD = 0x00f000f0u;
        const uint32_t v0 = w0[J] >> 8, v1 = w1[J] >> 8;
        ptx::mma_f16_16816(ca, w0[J] & EVEN, w1[J] & EVEN, v0 & EVEN, v1 & EVEN, f.qb[J][0], f.qb[J][2]);
        ptx::mma_f16_16816(cb, w0[J] & ODD, w1[J] & ODD, v0 & ODD, v1 & ODD, f.qb[J][1], f.qb[J][3]);
      }
    }
    constexpr float W = RAW ? 1.f : 0.0625f;  // of cb
    s[tile][0] = fmaf(sk0, fmaf(cb[0], W, ca[0]), qa.x);
    s[tile][1] = fmaf(sk0, fmaf(cb[1], W, ca[1]), qa.y);
    s[tile][2] = fmaf(sk1, fmaf(cb[2], W, ca[2]), qa.x);
    s[tile][3] = fmaf(sk1, fmaf(cb[3], W, ca[3]), qa.y);
    if (MASK) {
      // tokens past the end: score -inf (their buffer bytes are stale)
      if (tb + g >= nvalid) s[tile][0] = s[tile][1] = -INFINITY;
      if (tb + g + 8 >= nvalid) s[tile][2] = s[tile][3] = -INFINITY;
    }
    if (MASK == 2) {
      if (tb + g < vlo) s[tile][0] = s[tile][1] = -INFINITY;
      if (tb + g + 8 < vlo) s[tile][2] = s[tile][3] = -INFINITY;
    }
  }
  // ---------------- online softmax (base 2), lazy rescale
  bool moved = false;
  {
    float mx0 = fmaxf(s[0][0], s[0][2]), mx1 = fmaxf(s[0][1], s[0][3]);
#pragma unroll
    for (int tile = 1; tile < NT; ++tile) {
      mx0 = fmaxf(mx0, fmaxf(s[tile][0], s[tile][2]));
      mx1 = fmaxf(mx1, fmaxf(s[tile][1], s[tile][3]));
    }
    const bool need = (mx0 > st.m[0] + TAU) || (mx1 > st.m[1] + TAU);
    if (__any_sync(0xffffffffu, need)) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, o));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, o));
      }
      const float n0 = fmaxf(st.m[0], mx0), n1 = fmaxf(st.m[1], mx1);
      const float f0 = (n0 == -INFINITY) ? 1.f : fast_exp2(st.m[0] - n0);
      const float f1 = (n1 == -INFINITY) ? 1.f : fast_exp2(st.m[1] - n1);
      st.m[0] = n0;
      st.m[1] = n1;
      st.l[0] *= f0;
      st.l[1] *= f1;
      st.vb[0] *= f0;
      st.vb[1] *= f1;
      st.vb[2] *= f0;
      st.vb[3] *= f1;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        st.o[i][0] *= f0;
        st.o[i][1] *= f1;
        st.o[i][2] *= f0;
        st.o[i][3] *= f1;
      }
      // the factor of head g (the operand layout's head) for the chunk's earlier P
      const float a = __shfl_sync(0xffffffffu, f0, g >> 1), b = __shfl_sync(0xffffffffu, f1, g >> 1);
      fh = __float2half2_rn((g & 1) ? b : a);
      moved = true;
    }
  }
#pragma unroll
  for (int tile = 0; tile < NT; ++tile) {
    // masked scores are -inf and the running max is finite here: ex2(-inf) = 0
    const float p0 = fast_exp2(s[tile][0] - st.m[0]);
    const float p1 = fast_exp2(s[tile][1] - st.m[1]);
    const float p2 = fast_exp2(s[tile][2] - st.m[0]);
    const float p3 = fast_exp2(s[tile][3] - st.m[1]);
    if (!G::SPLIT) {  // 64-token chunks sum P through the indicator MMA's all-ones row instead
      st.l[0] += p0 + p2;
      st.l[1] += p1 + p3;
    }
    bp[tile] = make_uint2(ptx::movmatrix_trans(ptx::pack_half2(p0, p1)), ptx::movmatrix_trans(ptx::pack_half2(p2, p3)));
  }
  return moved;
}

// Output of the 16-token tile at chunk-local token tb with its P (bP0, bP1).
template <class G, int MASK>
__device__ __forceinline__ void v_tile(WarpState &st, const VAddr &A, int tb, uint32_t bP0, uint32_t bP1, int nvalid,
                                       int lane, int vlo = 0) {
  constexpr int lsv = G::LSV;
  // P' = P * scale_v: in the operand layout a lane holds tokens 2t, 2t+1 (and
  // 2t+8, 2t+9) of head g, whose V scales are one 32-bit word each
  uint32_t sw0 = ptx::lds_u32(A.scV + tb * 2), sw1 = ptx::lds_u32(A.scV + (tb + 8) * 2);
  if (MASK) {
    // scales past the end are stale bytes (P is 0 there, but 0 * inf is not)
    const int t2 = tb + 2 * (lane & 3);
    if (t2 >= nvalid) sw0 = 0u;
    else if (t2 + 1 >= nvalid) sw0 &= 0xffffu;
    if (t2 + 8 >= nvalid) sw1 = 0u;
    else if (t2 + 9 >= nvalid) sw1 &= 0xffffu;
    if (MASK == 2) {  // and so may the padding's be anything
      if (t2 + 1 < vlo) sw0 = 0u;
      else if (t2 < vlo) sw0 &= 0xffff0000u;
      if (t2 + 9 < vlo) sw1 = 0u;
      else if (t2 + 8 < vlo) sw1 &= 0xffff0000u;
    }
  }
  const uint32_t bS0 = ptx::h22u(__hmul2(ptx::u2h2(bP0), ptx::u2h2(sw0)));
  const uint32_t bS1 = ptx::h22u(__hmul2(ptx::u2h2(bP1), ptx::u2h2(sw1)));
  if (G::SPLIT) {
    // 64-token chunks have few V anchors (2 for stride 32): P is summed per
    // anchor slot of the chunk (rows of ps) by one MMA with an indicator
    // matrix (row a, token k: 1 when token k belongs to anchor a), and the
    // anchors are applied once per chunk (apply_v_anchors) instead of gathered
    // for every token
    constexpr uint32_t ONE2 = 0x3C003C00u;
    const int gg = lane >> 2, t2 = 2 * (lane & 3);
    const int s0 = (tb + t2) >> lsv, s1 = (tb + t2 + 8) >> lsv;
    const uint32_t r15 = gg == 7 ? ONE2 : 0u;  // row 15: every token (the softmax denominator)
    ptx::mma_f16_16816(st.ps, gg == s0 ? ONE2 : 0u, r15, gg == s1 ? ONE2 : 0u, r15, bP0, bP1);
  } else
  // V anchors: O += A_v^T P, ldmatrix.trans gathers each token's anchor row
  {
    uint32_t base = A.kfV + (uint32_t)((tb >> lsv) * (HD * 2));
    if (MASK) {
      // rows past the copied anchors hold stale bytes: use anchor 0 (P is 0 there)
      const int mi = lane >> 3, r = lane & 7;
      const int tok = tb + r + ((mi & 2) ? 8 : 0);
      if (MASK == 1 && tok >= nvalid) base = A.kfV0;
      // before vlo the anchors may be NaN: use the first counted token's
      if (MASK == 2 && (tok >= nvalid || tok < vlo)) base = A.kfV0 + (uint32_t)((vlo >> lsv) * (HD * 2));
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t a0, a1, a2, a3;
      ptx::ldmatrix_x4_trans(a0, a1, a2, a3, base + i * 32);
      ptx::mma_f16_16816(st.o[i], a0, a1, a2, a3, bP0, bP1);
    }
  }
  if constexpr (G::PL) {
    // bit-plane V codes: a row's low plane word g holds dims 8k + g (k = 0..15) at bits 2k; with
    // 3-bit codes a high plane half-word g holds the same dims' third bits at bit k
    // (CQ_ORDER_PLANES3, CQ_ORDER_PLANES2).  The fp16 operand 64 + v (v = code + 4, or code + 2)
    // gets the low bits at bits 4-5 and the high bit at bit 6 of each half
    constexpr uint32_t R = G::VR;  // bytes per row
    const int g = lane >> 2;
    const uint32_t r0 = A.cdV + (uint32_t)((tb - (tb >> lsv)) * R);
    const uint32_t r2 = r0 + (uint32_t)A.dv8 * R;
    const uint32_t lo = 4 * g, hi = 32 + 2 * g;
    const uint32_t la = ptx::lds_u32(r0 + lo), lb = ptx::lds_u32(r0 + R + lo);
    const uint32_t lc = ptx::lds_u32(r2 + lo), ld = ptx::lds_u32(r2 + R + lo);
    uint32_t hab = 0u, hcd = 0u;
    if constexpr (G::V3) {
      hab = __byte_perm(ptx::lds_u16(r0 + hi), ptx::lds_u16(r0 + R + hi), 0x5410u);
      hcd = __byte_perm(ptx::lds_u16(r2 + hi), ptx::lds_u16(r2 + R + hi), 0x5410u);
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int bi = 2 * q + half;  // byte of the low plane (4 dims), nibble of the high plane
        const uint32_t sel = bi | (bi << 4) | ((4 + bi) << 8) | ((4 + bi) << 12);
        const uint32_t xab = __byte_perm(la, lb, sel), xcd = __byte_perm(lc, ld, sel);
        uint32_t xa[4], xc[4];
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          const int sl = 4 - 2 * kk;  // low bits 2kk..2kk+1 -> 4..5; high bit kk -> 6
          const uint32_t pa = sl >= 0 ? xab << sl : xab >> -sl, pc = sl >= 0 ? xcd << sl : xcd >> -sl;
          xa[kk] = ptx::lop3_and_or(pa, 0x00300030u, 0x54005400u);
          xc[kk] = ptx::lop3_and_or(pc, 0x00300030u, 0x54005400u);
          if constexpr (G::V3) {
            const uint32_t yab = hab >> (4 * bi), ycd = hcd >> (4 * bi);
            xa[kk] = ptx::lop3_and_or(yab << (6 - kk), 0x00400040u, xa[kk]);
            xc[kk] = ptx::lop3_and_or(ycd << (6 - kk), 0x00400040u, xc[kk]);
          }
        }
        // dim index k = 8q + 4 half + kk <-> m-tile 4q + (4 half + kk)/2, row g (+8 when kk is odd)
        const int i0 = 4 * q + 2 * half;
        ptx::mma_f16_16816(st.o[i0], xa[0], xa[1], xc[0], xc[1], bS0, bS1);
        ptx::mma_f16_16816(st.o[i0 + 1], xa[2], xa[3], xc[2], xc[3], bS0, bS1);
      }
    }
    // the offset of every code value (68 or 66): offset * sum_t P'_t, exactly as the MMAs above weight it
    constexpr uint32_t OFF = G::V3 ? ptx::HALF2_68 : ptx::HALF2_66;
    ptx::mma_f16_16816(st.vb, OFF, OFF, OFF, OFF, bS0, bS1);
  } else
  // V codes: O += C_v^T P'  (tokens 2t,2t+1 | 2t+8,2t+9; words 2g, 2g+1)
  {
    // V rows of tokens tb+2t, +1, +8, +9 (stride 8: the I-frame at tb+8 sits between)
    const uint32_t rv = A.cdV + (uint32_t)((tb - (tb >> lsv)) * 64);
    const uint32_t rv8 = rv + (uint32_t)A.dv8 * 64;
    const uint2 va = ptx::lds_u64(rv);
    const uint2 vb = ptx::lds_u64(rv + 64);
    const uint2 vc = ptx::lds_u64(rv8);
    const uint2 vd = ptx::lds_u64(rv8 + 64);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const uint32_t wa = q ? va.y : va.x, wb = q ? vb.y : vb.x;
      const uint32_t wc = q ? vc.y : vc.x, wd = q ? vd.y : vd.x;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t sel = half ? 0x7632u : 0x5410u;
        uint32_t xa[4], xc[4];
        ptx::nibbles_to_half2_64(__byte_perm(wa, wb, sel), xa);  // nibbles 4*half + 0..3 of tokens (a, b)
        ptx::nibbles_to_half2_64(__byte_perm(wc, wd, sel), xc);
        // nibble j of word q <-> m-tile 4q + j/2, row g (+8 when j is odd)
        const int i0 = 4 * q + 2 * half;
        ptx::mma_f16_16816(st.o[i0], xa[0], xa[1], xc[0], xc[1], bS0, bS1);
        ptx::mma_f16_16816(st.o[i0 + 1], xa[2], xa[3], xc[2], xc[3], bS0, bS1);
      }
    }
    // the offset 72 of every code value: 72 * sum_t P'_t, exactly as the MMAs above weight it
    ptx::mma_f16_16816(st.vb, ptx::HALF2_72, ptx::HALF2_72, ptx::HALF2_72, ptx::HALF2_72, bS0, bS1);
  }
}

// O += A_v^T PS of a chunk whose P was summed per V anchor (SPLIT geometries), and
// the chunk's sum of P into the denominator.  row: the anchor row of slot lane & 7
// (slots out of use have weight 0: any row in use).
__device__ __forceinline__ void apply_v_anchors(WarpState &st, uint32_t row, int lane) {
  const uint32_t b0 = ptx::movmatrix_trans(ptx::pack_half2(st.ps[0], st.ps[1]));
  st.l[0] += st.ps[2];  // row 15 (lanes g == 7): this chunk's sum of P per head
  st.l[1] += st.ps[3];
  st.ps[0] = st.ps[1] = st.ps[2] = st.ps[3] = 0.f;
  const uint32_t base = row + (lane >> 3) * 16;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t a0, a1, a2, a3;
    ptx::ldmatrix_x4_trans(a0, a1, a2, a3, base + i * 64);
    ptx::mma_f16_16816(st.o[2 * i], a0, a1, 0u, 0u, b0, 0u);
    ptx::mma_f16_16816(st.o[2 * i + 1], a2, a3, 0u, 0u, b0, 0u);
  }
}

// Write the warp's state for one unit (its G real heads only) as a partial --
// max, sum and unnormalised output at pm[h], pl[h], po[h * HD + dim] -- and
// reset it.
__device__ __forceinline__ void flush_to(int G, WarpState &st, float *pm, float *pl, float *po, int lane) {
  const int g = lane >> 2, t = lane & 3;
  float l0 = st.l[0], l1 = st.l[1];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) st.o[i][j] -= st.vb[j];  // codes were 64 + n = (n - 8) + 72
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, o);
    l1 += __shfl_xor_sync(0xffffffffu, l1, o);
  }
  const int h0 = 2 * t, h1 = 2 * t + 1;
  if (g == 0) {
    if (h0 < G) {
      pm[h0] = st.m[0];
      pl[h0] = l0;
    }
    if (h1 < G) {
      pm[h1] = st.m[1];
      pl[h1] = l1;
    }
  }
  if (h0 < G) {
    float *w0 = po + h0 * HD;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w0[16 * i + g] = st.o[i][0];
      w0[16 * i + g + 8] = st.o[i][2];
    }
  }
  if (h1 < G) {
    float *w1 = po + h1 * HD;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w1[16 * i + g] = st.o[i][1];
      w1[16 * i + g + 8] = st.o[i][3];
    }
  }
  reset(st);
}

// ---------------------------------------------------------------------------
// host side: a geometry's numbers, and whether a cache is stored in it
// ---------------------------------------------------------------------------
struct GeoSpec {
  int sk, sv, vp, C, slot, buf;
  int off[6];  // K anchors, K codes, K scales, V anchors, V codes, V scales
};

template <class G>
inline GeoSpec geo_spec() {
  return GeoSpec{G::SK, G::SV, G::VP, G::C, G::SLOT, G::BUF,
                 {G::O_KF0, G::O_CD0, G::O_SC0, G::O_KF1, G::O_CD1, G::O_SC1}};
}

inline int v_pack_of(const cq_paged_cache &c) {
  return c.v.code_order == CQ_ORDER_PLANES3 ? 3 : c.v.code_order == CQ_ORDER_PLANES2 ? 2 : 4;
}

// The kernels read the chunk-block layout: per (page, head, chunk) one block
// [K anchors][K codes][K scales][V anchors][V codes][V scales] of the
// geometry, the six arrays' base pointers pointing into the first block; phs:
// bytes per (page, head).
inline bool stored_as(const cq_paged_cache &c, const GeoSpec &g, int64_t &phs) {
  if (c.page_tokens % g.C || c.k.chunk_tokens != g.C || c.v.chunk_tokens != g.C) return false;
  const cq_component *cc[2] = {&c.k, &c.v};
  const char *base = (const char *)c.k.keyframes;
  const int64_t cs = g.slot;
  phs = c.k.keyframe_head_stride * 2;
  for (int i = 0; i < 2; ++i) {
    const cq_component &k = *cc[i];
    if (k.keyframe_chunk_stride * 2 != cs || k.code_chunk_stride * 4 != cs || k.scale_chunk_stride * 2 != cs)
      return false;
    if (k.keyframe_head_stride * 2 != phs || k.code_head_stride * 4 != phs || k.scale_head_stride * 2 != phs)
      return false;
    if ((const char *)k.keyframes - base != g.off[3 * i] || (const char *)k.codes - base != g.off[3 * i + 1] ||
        (const char *)k.scales - base != g.off[3 * i + 2])
      return false;
  }
  return !(phs & 15) && phs >= cs * (c.page_tokens / g.C);
}

// The orders and alignment the kernels need, whatever the strides.
inline bool stored_for_mma(const cq_paged_cache &c) {
  if (c.head_dim != HD || c.k.code_order != CQ_ORDER_NATURAL) return false;
  if (c.v.code_order != CQ_ORDER_MMA && c.v.code_order != CQ_ORDER_PLANES3 && c.v.code_order != CQ_ORDER_PLANES2)
    return false;
  if (c.k.scale_index != CQ_SCALE_BY_TOKEN || c.v.scale_index != CQ_SCALE_BY_TOKEN) return false;
  return ((uintptr_t)c.k.keyframes & 15) == 0;
}

}  // namespace fast
}  // namespace cq
