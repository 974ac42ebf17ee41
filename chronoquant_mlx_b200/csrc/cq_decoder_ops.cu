// cq_decoder_ops.cu -- the elementwise steps of the decoder that drives the
// compressed cache end to end (bench config 5), fused so that a decode
// step is a handful of kernels per layer instead of dozens of small ones:
//
//   cq_rmsnorm        y = bf16(x * rsqrt(mean(x^2) + eps)) * w        (per row)
//   cq_qk_norm_rope   per head of a fused QKV row: RMSNorm over head_dim
//                     (q and k), then rotate-half RoPE at one position;
//                     q, k, v written as contiguous [B][H][D]
//   cq_silu_mul       y = bf16(silu(g)) * u                          (SwiGLU)
//   cq_qk_norm_rope_rows  the head norm and rotation for any number of tokens,
//                     each at its own position (prompts, ragged batches), q and
//                     k written head-major [B][H][S][D]
//
// The first three keep the rounding points of the equivalent torch expression in
// bf16/fp16: products in fp32, one rounding to the tensor dtype after each
// torch op.  Only the order of the fp32 sum of squares differs from torch's
// reduction, so a value can land one dtype ulp away.
#include "cq_common.cuh"
#include "cq_launch.cuh"
#include "cq_ptx.cuh"

namespace cq {
namespace dec {

__device__ __forceinline__ float ld(const void *p, int64_t i, int dt) { return load_as_float(p, i, dt); }
__device__ __forceinline__ float rnd(float x, int dt) { return round_dt(x, dt); }

// one block per row, 256 threads
__global__ void __launch_bounds__(256) rmsnorm_kernel(const void *x, const void *w, void *y, int dim, float eps,
                                                      int dt) {
  const int64_t row = blockIdx.x;
  const int64_t base = row * dim;
  float ss = 0.f;
  for (int i = threadIdx.x; i < dim; i += 256) {
    const float v = ld(x, base + i, dt);
    ss = fmaf(v, v, ss);
  }
  __shared__ float red[8];
  ss = warp_sum(ss);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
  __syncthreads();
  if (threadIdx.x < 32) {
    float t = threadIdx.x < 8 ? red[threadIdx.x] : 0.f;
    t = warp_sum(t);
    if (threadIdx.x == 0) red[0] = t;
  }
  __syncthreads();
  const float r = rsqrtf(red[0] / (float)dim + eps);
  for (int i = threadIdx.x; i < dim; i += 256) {
    const float n = rnd(ld(x, base + i, dt) * r, dt);            // (x * rsqrt(...)).to(dtype)
    store_from_float(y, base + i, n * ld(w, i, dt), dt);         // * w  (one rounding)
  }
}

// one warp per (row b, head h) of the fused QKV row: heads [0, Hq) are q,
// [Hq, Hq+Hkv) k, [Hq+Hkv, Hq+2Hkv) v.  head_dim 128: lane l holds dims
// 4l..4l+3, the rotate-half partner of dim i < 64 is i + 64 (lane l ^ 16).
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(const void *qkv, int64_t row_stride, int B, int Hq, int Hkv,
                                                           const void *wq, const void *wk, const float *inv_freq,
                                                           const int64_t *pos, float eps, void *q_out, void *k_out,
                                                           void *v_out, int dt) {
  const int64_t gw = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  const int H = Hq + 2 * Hkv;
  if (gw >= (int64_t)B * H) return;
  const int b = (int)(gw / H), h = (int)(gw - (int64_t)b * H);
  constexpr int D = 128;
  const int64_t src = (int64_t)b * row_stride + (int64_t)h * D + 4 * lane;
  float x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = ld(qkv, src + i, dt);
  if (h >= Hq + Hkv) {  // v: copied
    const int64_t dst = ((int64_t)b * Hkv + (h - Hq - Hkv)) * D + 4 * lane;
#pragma unroll
    for (int i = 0; i < 4; ++i) store_from_float(v_out, dst + i, x[i], dt);
    return;
  }
  const bool is_q = h < Hq;
  const void *w = is_q ? wq : wk;
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) ss = fmaf(x[i], x[i], ss);
  ss = warp_sum(ss);
  const float r = rsqrtf(ss / (float)D + eps);
  float n[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) n[i] = rnd(rnd(x[i] * r, dt) * ld(w, 4 * lane + i, dt), dt);  // RMSNorm as above
  const float p = (float)*pos;
  const bool lo = lane < 16;
  float out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float partner = __shfl_xor_sync(0xffffffffu, n[i], 16);
    const int d = 4 * lane + i;
    const float ang = p * inv_freq[d & 63];
    const float rot = lo ? rnd(-partner, dt) : partner;  // cat(-x[64:], x[:64])
    out[i] = __fadd_rn(__fmul_rn(n[i], cosf(ang)), __fmul_rn(rot, sinf(ang)));  // x*cos + rot*sin, unfused
  }
  const int64_t dst = is_q ? ((int64_t)b * Hq + h) * D + 4 * lane : ((int64_t)b * Hkv + (h - Hq)) * D + 4 * lane;
  void *o = is_q ? q_out : k_out;
#pragma unroll
  for (int i = 0; i < 4; ++i) store_from_float(o, dst + i, out[i], dt);
}

// Head norm and rotation of many tokens.  The angle of a channel pair is pos *
// inv_freq in fp64 as a product and what its rounding left off (a product of two
// fp32 numbers is off by radians at far positions, one rounded to fp64 by 6e-5 at
// 2^40), reduced to [-pi, pi] there; its sine and cosine are shared by the
// token's heads.  All arithmetic is fp32 with one rounding to the tensor type at
// the end.
struct RopeArgs {
  const void *qkv;
  int64_t sb, ss;        // element strides of a sequence and a token
  int B, S, Hq, Hkv, D, rot, adjacent;
  const void *wq, *wk;   // both null: rotation only
  const float *inv_freq;
  const int64_t *pos;
  int64_t p_sb, p_ss;
  float eps;
  void *q_out, *k_out;
};

constexpr int kRopeWarps = 8;

// (cos, sin) of pair i at position p, exact to fp32 for |p| <= 2^53 (larger ones round to a double themselves) and
// |inv_freq| <= 1.
__device__ __forceinline__ float2 rope_angle(int64_t p, float inv_freq) {
  const double pd = (double)p, f = (double)inv_freq, ang = pd * f, rest = fma(pd, f, -ang);
  // 2 pi as the sum of two doubles (Cody and Waite's reduction): ang - n hi is a double's few last bits for the n
  // next to ang / hi, n lo is below 0.4, and what lo leaves off of 2 pi (below 2^-106) times n stays below 2^-54
  const double hi = 6.283185307179586, lo = 2.4492935982947064e-16;
  const double n = rint(ang * (1.0 / hi));
  const double r = fma(-n, lo, fma(-n, hi, ang)) + rest;
  float sn, cs;
  sincospif((float)(r * (2.0 / hi)), &sn, &cs);  // of r = pi x: no reduction left to do
  return make_float2(cs, sn);
}

// Four consecutive channels in one access (the addresses are 4 elements aligned).
template <int DT>
struct Quad {
  using Raw = uint2;
};
template <>
struct Quad<CQ_F32> {
  using Raw = uint4;
};
template <int DT>
__device__ __forceinline__ typename Quad<DT>::Raw load_quad(const void *p, int64_t i) {
  using R = typename Quad<DT>::Raw;
  return *(const R *)((const char *)p + i * (int64_t)(sizeof(R) / 4));
}
template <int DT>
__device__ __forceinline__ float4 widen(const typename Quad<DT>::Raw &u) {
  if constexpr (DT == CQ_F32) {
    return make_float4(__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w));
  } else {
    float2 a, b;
    if constexpr (DT == CQ_F16) {
      a = __half22float2(*(const __half2 *)&u.x);
      b = __half22float2(*(const __half2 *)&u.y);
    } else {
      a = __bfloat1622float2(*(const __nv_bfloat162 *)&u.x);
      b = __bfloat1622float2(*(const __nv_bfloat162 *)&u.y);
    }
    return make_float4(a.x, a.y, b.x, b.y);
  }
}
template <int DT>
__device__ __forceinline__ void store_quad(void *p, int64_t i, const float4 v) {
  if constexpr (DT == CQ_F32) {
    *(float4 *)((float *)p + i) = v;
  } else if constexpr (DT == CQ_F16) {
    const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
    *(uint2 *)((uint16_t *)p + i) = make_uint2(*(const uint32_t *)&a, *(const uint32_t *)&b);
  } else {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *(uint2 *)((uint16_t *)p + i) = make_uint2(*(const uint32_t *)&a, *(const uint32_t *)&b);
  }
}

// D / 8 lanes hold a head, each two quads of channels that rotate with each
// other: with halves, lane l < rot/8 the quads at 4l and rot/2 + 4l; with
// adjacent pairs, 8l and 8l + 4; lanes past the rotated channels take theirs in
// order and keep them.  So a head needs no exchange between lanes but the sum of
// squares.  A CTA takes TILE tokens; each group of lanes keeps one token, works out
// its lanes' four angles (no exchange, no barrier) and walks its share of the
// query heads, then of the key heads, UN heads' loads in flight, with the
// products of norm weight and sine or cosine in registers: a pair (x, y) of a
// head with root r becomes r (x wc - y ws'), r (y wc' + x ws).  Neighbouring
// groups hold neighbouring tokens, whose output rows are contiguous.  Bound by
// HBM: 2 x 8191 tokens of 32 + 8 + 8 bf16 heads of 128 (336 MB) take 60.9 us, 85 %
// of the measured copy rate; with two or eight heads in flight 66 and 67 us.
struct PairTurn {  // coefficients of one pair: out0 = x * xc - y * ys, out1 = y * yc + x * xs
  float xc, ys, yc, xs;
};

template <int DT, int D, int TILE>
__global__ void __launch_bounds__(kRopeWarps * 32, DT == CQ_F32 ? 3 : 4) qk_norm_rope_quads_kernel(RopeArgs A) {
  constexpr int LPH = D / 8, groups = kRopeWarps * 32 / LPH, DH = groups / TILE, UN = 4;
  using Raw = typename Quad<DT>::Raw;
  constexpr int ES = sizeof(Raw) / 4, ISTEP = DH * D * ES;  // bytes between two of a group's heads in a row
  ptx::grid_dependency_wait();
  const unsigned tok0 = blockIdx.x * TILE, n_tok = (unsigned)A.B * (unsigned)A.S;  // below 2^31
  const int half = A.rot / 2;
  const int l = threadIdx.x & (LPH - 1), group = threadIdx.x / LPH;
  const int tt = group & (TILE - 1), h0 = group / TILE;
  const bool turns = l < A.rot / 8, halves = !A.adjacent && turns, live = tok0 + tt < n_tok;
  const int da = halves ? 4 * l : 8 * l, db = halves ? half + 4 * l : 8 * l + 4;
  const unsigned tok = min(tok0 + tt, n_tok - 1), b = tok / (unsigned)A.S, s = tok - b * (unsigned)A.S;
  float2 cs[4];  // (cos, sin) of the lane's four pairs
#pragma unroll
  for (int i = 0; i < 4; ++i) cs[i] = make_float2(1.f, 0.f);
#pragma unroll 1
  for (int part = (int)blockIdx.y; part < 2; part += (int)gridDim.y) {  // query heads, then key heads (or a CTA each)
    const int H = part ? A.Hkv : A.Hq;
    const char *in = (const char *)A.qkv + (b * A.sb + s * A.ss + (int64_t)((part ? A.Hq : 0) + h0) * D) * ES;
    const char *ia = in + da * ES, *ib = in + db * ES;
    const int64_t row = (int64_t)A.S * D * ES, ostep = DH * row;
    char *out = (char *)(part ? A.k_out : A.q_out) + ((int64_t)b * H + h0) * row + (int64_t)s * (D * ES);
    char *oa = out + da * ES, *ob = out + db * ES;
    Raw ra[UN], rc[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u)
      if (h0 + u * DH < H) {
        ra[u] = *(const Raw *)(ia + u * ISTEP);
        rc[u] = *(const Raw *)(ib + u * ISTEP);
      } else {
        ra[u] = rc[u] = Raw{};
      }
    if (part == (int)blockIdx.y && turns) {  // under the first loads' latency
      const int64_t at = A.pos[b * A.p_sb + s * A.p_ss];
#pragma unroll
      for (int i = 0; i < 4; ++i) cs[i] = rope_angle(at, A.inv_freq[4 * l + i]);
    }
    PairTurn p[4];
    {
      const void *w = part ? A.wk : A.wq;
      float4 wa = make_float4(1.f, 1.f, 1.f, 1.f), wb = wa;
      if (w) wa = widen<DT>(load_quad<DT>(w, da)), wb = widen<DT>(load_quad<DT>(w, db));
      auto turn = [](float wx, float wy, float2 a) { return PairTurn{wx * a.x, wy * a.y, wy * a.x, wx * a.y}; };
      if (!A.adjacent) {  // pairs (a.i, c.i)
        p[0] = turn(wa.x, wb.x, cs[0]);
        p[1] = turn(wa.y, wb.y, cs[1]);
        p[2] = turn(wa.z, wb.z, cs[2]);
        p[3] = turn(wa.w, wb.w, cs[3]);
      } else {  // pairs (a.x, a.y) (a.z, a.w) (c.x, c.y) (c.z, c.w)
        p[0] = turn(wa.x, wa.y, cs[0]);
        p[1] = turn(wa.z, wa.w, cs[1]);
        p[2] = turn(wb.x, wb.y, cs[2]);
        p[3] = turn(wb.z, wb.w, cs[3]);
      }
    }
    for (int base = 0; base < H; base += DH * UN) {  // the same trips for every lane: the sums are shuffles
      ia += UN * ISTEP;
      ib += UN * ISTEP;
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        const int h = base + h0 + u * DH;
        const float4 a = widen<DT>(ra[u]), c = widen<DT>(rc[u]);
        if (h + DH * UN < H) {  // this slot's next head
          ra[u] = *(const Raw *)(ia + u * ISTEP);
          rc[u] = *(const Raw *)(ib + u * ISTEP);
        }
        float r = 1.f;
        if (A.wq) {
          float sq = a.x * a.x, s2 = c.x * c.x;
          sq = fmaf(a.y, a.y, sq);
          s2 = fmaf(c.y, c.y, s2);
          sq = fmaf(a.z, a.z, sq);
          s2 = fmaf(c.z, c.z, s2);
          sq = fmaf(a.w, a.w, sq);
          s2 = fmaf(c.w, c.w, s2);
          sq += s2;
#pragma unroll
          for (int o = 1; o < LPH; o <<= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
          r = rsqrtf(fmaf(sq, 1.f / D, A.eps));
        }
        float4 x, y;
        auto pair = [&](const PairTurn &t, float u0, float u1, float &o0, float &o1) {
          o0 = (u0 * t.xc - u1 * t.ys) * r;
          o1 = (u1 * t.yc + u0 * t.xs) * r;
        };
        if (!turns) {  // channels past the rotated ones, alone (no product with their neighbours)
          if (!A.adjacent) {
            x = make_float4(a.x * p[0].xc * r, a.y * p[1].xc * r, a.z * p[2].xc * r, a.w * p[3].xc * r);
            y = make_float4(c.x * p[0].yc * r, c.y * p[1].yc * r, c.z * p[2].yc * r, c.w * p[3].yc * r);
          } else {
            x = make_float4(a.x * p[0].xc * r, a.y * p[0].yc * r, a.z * p[1].xc * r, a.w * p[1].yc * r);
            y = make_float4(c.x * p[2].xc * r, c.y * p[2].yc * r, c.z * p[3].xc * r, c.w * p[3].yc * r);
          }
        } else if (!A.adjacent) {
          pair(p[0], a.x, c.x, x.x, y.x);
          pair(p[1], a.y, c.y, x.y, y.y);
          pair(p[2], a.z, c.z, x.z, y.z);
          pair(p[3], a.w, c.w, x.w, y.w);
        } else {
          pair(p[0], a.x, a.y, x.x, x.y);
          pair(p[1], a.z, a.w, x.z, x.w);
          pair(p[2], c.x, c.y, y.x, y.y);
          pair(p[3], c.z, c.w, y.z, y.w);
        }
        if (h < H && live) {
          store_quad<DT>(oa, 0, x);
          store_quad<DT>(ob, 0, y);
        }
        oa += ostep;
        ob += ostep;
      }
    }
  }
}

// Every other shape (head sizes that are no 64, 128 or 256, rotations that end
// inside a quad, rows off the quads' alignment): one CTA per token, a warp per
// head in turn, channels exchanged through shared memory.
template <int DT>
__global__ void __launch_bounds__(kRopeWarps * 32) qk_norm_rope_rows_kernel(RopeArgs A) {
  __shared__ float2 s_cs[128];              // (cos, sin) of each pair
  __shared__ float s_x[kRopeWarps][256];    // a head's normalised channels
  ptx::grid_dependency_wait();
  const int64_t tok = blockIdx.x;
  const int b = (int)(tok / A.S), s = (int)(tok - (int64_t)b * A.S);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int half = A.rot / 2, D = A.D, H = A.Hq + A.Hkv;
  for (int i = threadIdx.x; i < half; i += blockDim.x)
    s_cs[i] = rope_angle(A.pos[b * A.p_sb + s * A.p_ss], A.inv_freq[i]);
  __syncthreads();
  float *x = s_x[warp];
  for (int h = warp; h < H; h += kRopeWarps) {
    const int64_t src = b * A.sb + s * A.ss + (int64_t)h * D;
    const void *w = h < A.Hq ? A.wq : A.wk;
    float v[8], sq = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int d = lane + 32 * k;
      v[k] = d < D ? load_as_float(A.qkv, src + d, DT) : 0.f;
      sq = fmaf(v[k], v[k], sq);
    }
    const float r = w ? rsqrtf(warp_sum(sq) / (float)D + A.eps) : 1.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int d = lane + 32 * k;
      if (d < D) x[d] = w ? v[k] * r * load_as_float(w, d, DT) : v[k];
    }
    __syncwarp();
    const bool is_q = h < A.Hq;
    void *out = is_q ? A.q_out : A.k_out;
    const int64_t dst = is_q ? (((int64_t)b * A.Hq + h) * A.S + s) * D
                             : (((int64_t)b * A.Hkv + (h - A.Hq)) * A.S + s) * D;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int d = lane + 32 * k;
      if (d >= D) continue;
      float y = x[d];
      if (d < A.rot) {
        const int i = A.adjacent ? d >> 1 : (d < half ? d : d - half);
        const bool second = A.adjacent ? (d & 1) : d >= half;
        const float o = x[A.adjacent ? d ^ 1 : (second ? d - half : d + half)];
        const float2 cs = s_cs[i];
        y = second ? fmaf(y, cs.x, o * cs.y) : fmaf(y, cs.x, -o * cs.y);
      }
      store_from_float(out, dst + d, y, DT);
    }
    __syncwarp();
  }
}

// gu: [rows][2*ffn] (gate | up); y: [rows][ffn]
__global__ void silu_mul_kernel(const void *gu, void *y, int64_t rows, int ffn, int dt) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= rows * ffn) return;
  const int64_t r = i / ffn, c = i - r * ffn;
  const float g = ld(gu, r * 2 * ffn + c, dt), u = ld(gu, r * 2 * ffn + ffn + c, dt);
  const float s = rnd(g / (1.f + expf(-g)), dt);  // silu(g) in the tensor dtype
  store_from_float(y, i, s * u, dt);
}

}  // namespace dec
}  // namespace cq

using namespace cq;

extern "C" int cq_rmsnorm(const void *x, const void *w, void *y, int64_t rows, int32_t dim, float eps, int dtype,
                          void *stream) {
  CQ_REQUIRE(x && w && y && rows >= 0 && dim >= 1, CQ_ERR_INVALID, "cq_rmsnorm: bad arguments");
  CQ_REQUIRE(dtype == CQ_F16 || dtype == CQ_BF16, CQ_ERR_UNSUPPORTED, "cq_rmsnorm: dtype must be f16/bf16");
  if (rows == 0) return CQ_OK;
  CQ_REQUIRE(rows < (1LL << 31), CQ_ERR_INVALID, "cq_rmsnorm: too many rows");
  dec::rmsnorm_kernel<<<(unsigned)rows, 256, 0, (cudaStream_t)stream>>>(x, w, y, dim, eps, dtype);
  return check_launch("cq_rmsnorm");
}

extern "C" int cq_qk_norm_rope(const void *qkv, int64_t row_stride, int32_t batch, int32_t n_q_heads,
                               int32_t n_kv_heads, int32_t head_dim, const void *q_norm_w, const void *k_norm_w,
                               const float *inv_freq, const int64_t *pos, float eps, void *q_out, void *k_out,
                               void *v_out, int dtype, void *stream) {
  CQ_REQUIRE(qkv && q_norm_w && k_norm_w && inv_freq && pos && q_out && k_out && v_out, CQ_ERR_INVALID,
             "cq_qk_norm_rope: null pointer");
  CQ_REQUIRE(head_dim == 128, CQ_ERR_UNSUPPORTED, "cq_qk_norm_rope: head_dim must be 128");
  CQ_REQUIRE(dtype == CQ_F16 || dtype == CQ_BF16, CQ_ERR_UNSUPPORTED, "cq_qk_norm_rope: dtype must be f16/bf16");
  CQ_REQUIRE(batch >= 1 && n_q_heads >= 1 && n_kv_heads >= 1, CQ_ERR_INVALID, "cq_qk_norm_rope: bad sizes");
  const int64_t warps = (int64_t)batch * (n_q_heads + 2 * n_kv_heads);
  dec::qk_norm_rope_kernel<<<(unsigned)((warps + 7) / 8), 256, 0, (cudaStream_t)stream>>>(
      qkv, row_stride, batch, n_q_heads, n_kv_heads, q_norm_w, k_norm_w, inv_freq, pos, eps, q_out, k_out, v_out,
      dtype);
  return check_launch("cq_qk_norm_rope");
}

extern "C" int cq_silu_mul(const void *gu, void *y, int64_t rows, int32_t ffn, int dtype, void *stream) {
  CQ_REQUIRE(gu && y && rows >= 0 && ffn >= 1, CQ_ERR_INVALID, "cq_silu_mul: bad arguments");
  CQ_REQUIRE(dtype == CQ_F16 || dtype == CQ_BF16, CQ_ERR_UNSUPPORTED, "cq_silu_mul: dtype must be f16/bf16");
  const int64_t n = rows * ffn;
  if (n == 0) return CQ_OK;
  CQ_REQUIRE((n + 255) / 256 < (1LL << 31), CQ_ERR_INVALID, "cq_silu_mul: too large");
  dec::silu_mul_kernel<<<(unsigned)((n + 255) / 256), 256, 0, (cudaStream_t)stream>>>(gu, y, rows, ffn, dtype);
  return check_launch("cq_silu_mul");
}

extern "C" int cq_qk_norm_rope_rows(const void *qkv, int64_t seq_stride, int64_t row_stride, int32_t batch,
                                    int32_t tokens, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                                    int32_t rot_dim, int32_t adjacent, const void *q_norm_w, const void *k_norm_w,
                                    const float *inv_freq, const int64_t *pos, int64_t pos_sb, int64_t pos_ss,
                                    float eps, void *q_out, void *k_out, int dtype, void *stream) {
  CQ_REQUIRE((q_norm_w == nullptr) == (k_norm_w == nullptr), CQ_ERR_INVALID,
             "cq_qk_norm_rope_rows: give both norm weights or neither");
  CQ_REQUIRE(batch >= 0 && tokens >= 0 && n_q_heads >= 1 && n_kv_heads >= 1, CQ_ERR_INVALID,
             "cq_qk_norm_rope_rows: bad sizes");
  CQ_REQUIRE(n_q_heads < (1 << 20) && n_kv_heads < (1 << 20), CQ_ERR_UNSUPPORTED, "cq_qk_norm_rope_rows: too many heads");
  CQ_REQUIRE(head_dim >= 8 && head_dim <= 256 && head_dim % 8 == 0, CQ_ERR_UNSUPPORTED,
             "cq_qk_norm_rope_rows: head_dim must be a multiple of 8 in [8, 256]");
  CQ_REQUIRE(rot_dim >= 0 && rot_dim <= head_dim && rot_dim % 2 == 0, CQ_ERR_INVALID,
             "cq_qk_norm_rope_rows: rot_dim must be even and at most head_dim");
  CQ_REQUIRE(dtype == CQ_F16 || dtype == CQ_BF16 || dtype == CQ_F32, CQ_ERR_UNSUPPORTED,
             "cq_qk_norm_rope_rows: dtype must be f16, bf16 or f32");
  const int64_t n = (int64_t)batch * tokens;
  if (n == 0) return CQ_OK;
  CQ_REQUIRE(n < (1LL << 31), CQ_ERR_INVALID, "cq_qk_norm_rope_rows: too many tokens");
  CQ_REQUIRE(qkv && q_out && k_out, CQ_ERR_INVALID, "cq_qk_norm_rope_rows: null pointer");
  CQ_REQUIRE(rot_dim == 0 || (inv_freq && pos), CQ_ERR_INVALID, "cq_qk_norm_rope_rows: inv_freq or pos is null");
  const dec::RopeArgs A{qkv,      seq_stride, row_stride, batch, tokens, n_q_heads, n_kv_heads, head_dim, rot_dim, adjacent,
                        q_norm_w, k_norm_w,   inv_freq,   pos,   pos_sb, pos_ss,    eps,        q_out,    k_out};
  cudaStream_t st = (cudaStream_t)stream;
  // the quads need 4-element alignment of every row and of the weights, and a rotation that ends with a quad
  const uintptr_t unit = dtype == CQ_F32 ? 16 : 8, es = unit / 4;
  const bool quads = (head_dim == 64 || head_dim == 128 || head_dim == 256) && rot_dim % 8 == 0 &&
                     (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)q_norm_w |
                       (uintptr_t)k_norm_w | (uintptr_t)(seq_stride * (int64_t)es) |
                       (uintptr_t)(row_stride * (int64_t)es)) & (unit - 1)) == 0;
  if (quads) {
    // 8 tokens per CTA where there are CTAs enough (their rows are written next to each other), else one, its query
    // and key heads in CTAs of their own
    const bool tiled = n >= 8 * 2 * sm_count();
    const dim3 grid((unsigned)(tiled ? (n + 7) / 8 : n), tiled ? 1 : 2);
#define CQ_ROPE(DT)                                                                                         \
  (head_dim == 64    ? (tiled ? dec::qk_norm_rope_quads_kernel<DT, 64, 8> : dec::qk_norm_rope_quads_kernel<DT, 64, 1>)   \
   : head_dim == 128 ? (tiled ? dec::qk_norm_rope_quads_kernel<DT, 128, 8> : dec::qk_norm_rope_quads_kernel<DT, 128, 1>) \
                     : (tiled ? dec::qk_norm_rope_quads_kernel<DT, 256, 8> : dec::qk_norm_rope_quads_kernel<DT, 256, 1>))
    auto *fn = dtype == CQ_F16 ? CQ_ROPE(CQ_F16) : dtype == CQ_BF16 ? CQ_ROPE(CQ_BF16) : CQ_ROPE(CQ_F32);
#undef CQ_ROPE
    return launch_after(fn, grid, dec::kRopeWarps * 32, 0, st, "cq_qk_norm_rope_rows", A);
  }
  auto *fn = dtype == CQ_F16    ? dec::qk_norm_rope_rows_kernel<CQ_F16>
             : dtype == CQ_BF16 ? dec::qk_norm_rope_rows_kernel<CQ_BF16>
                                : dec::qk_norm_rope_rows_kernel<CQ_F32>;
  return launch_after(fn, dim3((unsigned)n), dec::kRopeWarps * 32, 0, st, "cq_qk_norm_rope_rows", A);
}
