// cq_sparse_fast.cu -- block-sparse attention on the chunk-block layout.
//
// A unit is one (sequence, kv-head, query token): the tokens of its listed
// blocks, cut into the cache's chunks (32 or 64 tokens, one contiguous block of
// bytes each), attended by every query head of the group.  W = w * s warps share
// a unit: w warps of a CTA, and with more than 8 of them s CTAs of a cluster.
// Warp r takes the list's chunk slots r, r + W, ...: its lanes look up 32 slots
// at once (list entry, page, visible tokens), the ones that hold a visible token
// are streamed with bulk copies and computed by the decode kernel's core
// (cq_decode_core.cuh: scores and output as MMAs on the packed codes).  The
// warps' partial (max, sum, output) are merged in shared memory, across the
// cluster through distributed shared memory: one launch, no workspace, and the
// order of every sum is fixed.
//
// Scores, maxima, sums and outputs are held in fp32.  Fewer bits where the tensor
// cores take fp16 operands, as in the decode kernel: q * scale (exact for queries
// of either type within fp16's normal range); P, up to 2^8 while the maximum lags
// (2^-11 relative); P times the token's V scale (2^-11 more, finite for scales
// below 256); P summed per V anchor in fp32 and rounded as the operand that weights
// the anchors; earlier P of a chunk times the correction when the maximum moves.
// With sum p = 1 an output stays within 5 * 2^-11 max|v| of the exact one; fp32
// operands (tf32 products) would halve the products' rate and double the buffers.
//
// Bound by latency where units are few (one query over 32 blocks of 64: 7.8 us)
// and by instructions where they are many: 4096 units of 32 chunks take 217 us,
// 1025 instructions a chunk of which half run on the half-rate integer pipe, at
// 58 % issue with the 16 warps an SM that registers and buffers leave room for.
// Each listed chunk is decoded once per query token that lists it (16 times on
// average over 512 tokens).  Several neighbouring tokens per unit, sharing the
// chunks that more than one of them lists, took 255 to 301 us (their lists overlap
// by a third).
//
// Requirements (sparse_fast_supported): the decode kernel's layouts, a GQA
// group of at most 8, block_tokens a multiple of the chunk.
#include <algorithm>
#include <mutex>
#include <string>

#include "cq_decode_core.cuh"
#include "cq_sparse.cuh"

namespace cq {
namespace fast {

constexpr int kSW = 8;            // warps per CTA (two CTAs per SM)
constexpr int kMaxCluster = 8;    // CTAs per unit
constexpr int kPartFloats = 16 + 8 * HD;  // a partial: [8] max, [8] sum, [8][HD] output

struct SparseParams {
  CacheView cv;
  const char *blk;
  int64_t phs;
  const void *q;
  int q_dtype;
  int64_t q_sb, q_sh, q_sq;
  float scale;
  int gqa, q_len, top, bt;
  int64_t T;
  const int64_t *len_dev, *starts;
  const int32_t *blocks;
  int cpb;        // chunks per block
  int w, s;       // warps per unit in a CTA, CTAs per unit
  unsigned units;
  void *out;
  int out_dtype;
  float *lse_out;
};

__device__ int g_sparse_fast_error;

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of this CTA's shared-memory word `a` in CTA `rank` of the cluster, and loads from there.
__device__ __forceinline__ uint32_t map_shared(uint32_t a, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}
__device__ __forceinline__ float ld_cluster(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(a)
               : "memory");
  return v;
}

// One part of a chunk's block at `src` (0: K part, 1: V part, 2: all of it), by one lane.
template <class G, int PART>
__device__ __forceinline__ void copy_part(uint32_t buf, uint64_t *bar, const char *src, int lane) {
  if (lane != 0) return;
  constexpr int off = PART == 1 ? G::O_KF1 : 0, bytes = PART == 2 ? G::SLOT : (PART ? G::VB : G::KB);
  ptx::mbar_arrive_expect_tx(bar, (uint32_t)bytes);
  ptx::bulk_g2s_a(buf, src + off, (uint32_t)bytes, bar);
}

// One chunk whose tokens [vlo, vhi) count; `next`: the block that follows in
// its buffers (null: none).  False when a wait gave up.
template <class G, int MASK>
__device__ __forceinline__ bool sparse_chunk(WarpState &st, const QFrag &f, int vlo, int vhi, unsigned char *region,
                                             uint64_t *bar, int sk, uint32_t ph, const char *next, float *qa,
                                             const unsigned char *qt, int lane) {
  constexpr int NG = G::NT / 2;  // 32-token groups
  const uint32_t ra = ptx::smem_u32(region);
  const uint32_t kb = ra + (G::SPLIT ? 0 : sk * G::SLOT), vb = ra + (G::SPLIT ? G::KB : sk * G::SLOT + G::O_KF1);
  if (!ptx::mbar_wait_bounded(&bar[sk], ph, WAIT_BUDGET)) return false;
  compute_qa_tile(kb + G::O_KF0, qa, MASK ? ((vhi - 1) >> G::LSK) + 1 : G::AK, qt, lane);
  __syncwarp();
  uint2 bp[NG][2];
  {
    const KAddr A(G(), kb, ptx::smem_u32(qa), lane);
#pragma unroll
    for (int grp = 0; grp < NG; ++grp) {
      if (MASK && (grp * 32 >= vhi || grp * 32 + 32 <= vlo)) continue;
      __half2 fh;
      if (k_group<G, MASK, false>(st, A, f, grp * 32, vhi, lane, bp[grp], fh, vlo)) {
#pragma unroll
        for (int k = 0; k < grp; ++k)
#pragma unroll
          for (int tile = 0; tile < 2; ++tile) {
            if (MASK && k * 32 + 32 <= vlo) continue;
            bp[k][tile].x = ptx::h22u(__hmul2(ptx::u2h2(bp[k][tile].x), fh));
            bp[k][tile].y = ptx::h22u(__hmul2(ptx::u2h2(bp[k][tile].y), fh));
          }
      }
    }
  }
  if (G::SPLIT) {
    __syncwarp();
    ptx::fence_proxy_async_smem();
    if (next) copy_part<G, 0>(kb, &bar[sk], next, lane);
    if (!ptx::mbar_wait_bounded(&bar[G::NSK + sk], ph, WAIT_BUDGET)) return false;
  }
  {
    const VAddr A(G(), vb, lane);
#pragma unroll
    for (int grp = 0; grp < NG; ++grp)
#pragma unroll
      for (int tile = 0; tile < 2; ++tile) {
        const int tb = grp * 32 + tile * 16;
        if (MASK && (tb >= vhi || tb + 16 <= vlo)) continue;
        v_tile<G, MASK>(st, A, tb, bp[grp][tile].x, bp[grp][tile].y, vhi, lane, vlo);
      }
    if (G::SPLIT) {  // rows of anchors that counted tokens use
      const int a0 = MASK ? vlo >> G::LSV : 0, a1 = MASK ? (vhi - 1) >> G::LSV : G::AV - 1;
      apply_v_anchors(st, vb + max(a0, min(lane & 7, a1)) * (HD * 2), lane);
    }
  }
  __syncwarp();
  ptx::fence_proxy_async_smem();
  if (next) {
    if (G::SPLIT)
      copy_part<G, 1>(vb, &bar[G::NSK + sk], next, lane);
    else
      copy_part<G, 2>(kb, &bar[sk], next, lane);
  }
  return true;
}

// The chunks of rank r of unit (b, h, i); the partial is left in `region`.
template <class G>
__device__ __forceinline__ void unit_main(const SparseParams &p, int64_t T, unsigned unit, int r, unsigned char *region,
                                          uint64_t *bar, int lane) {
  // positions and units in 32 bits (the launch keeps them there)
  const int W = p.w * p.s, n = p.top * p.cpb;
  const unsigned bh = unit / (unsigned)p.q_len;
  const int i = (int)(unit - bh * (unsigned)p.q_len);
  const int b = (int)(bh / (unsigned)p.cv.H), h = (int)(bh - (unsigned)b * (unsigned)p.cv.H);
  const int pos = (int)T - p.q_len + i, st0 = (int)min(sparse::first_token(p.starts, b), (int64_t)INT32_MAX);
  const int last = (int)((unsigned)pos / (unsigned)p.bt);  // the query's own block
  const int32_t *list = p.blocks + (int64_t)unit * p.top;
  const uint32_t ra = ptx::smem_u32(region);
  float *qa = (float *)(region + G::BUF);
  unsigned char *qt = region + G::BUF + kQaBytes;
  WarpState st;
  reset(st);
  QFrag f;
  bool have_q = false;
  int sk = 0;
  uint32_t ph = 0;
  for (int base = r; base < n; base += 32 * W) {
    // 32 chunk slots at once, one per lane: where the chunk's block lies and which of its tokens count
    const char *src = nullptr;
    int vlo = 0, vhi = 0;
    const int64_t x = base + (int64_t)lane * W;
    if (x < n) {
      const int slot = (int)x / p.cpb, c = (int)x - slot * p.cpb;
      const int j = list[slot];
      if (j >= 0 && j <= last && (slot == 0 || j > list[slot - 1])) {
        const int t0 = j * p.bt + c * G::C;
        const int lo = max(0, st0 - t0), hi = min(G::C, pos + 1 - t0);
        if (lo < hi) {
          const int lp = (int)((unsigned)t0 / (unsigned)p.cv.P);
          const int jc = (t0 - lp * p.cv.P) / G::C;
          src = p.blk + (table_page(p.cv, b, lp) * p.cv.H + h) * p.phs + (int64_t)jc * G::SLOT;
          vlo = lo;
          vhi = hi;
        }
      }
    }
    unsigned todo = __ballot_sync(0xffffffffu, vhi > 0), issue = todo;
    auto take = [&](unsigned &m) -> const char * {  // the next block of the mask, null when it is empty
      const int l = m ? __ffs(m) - 1 : 0;
      const char *a = (const char *)__shfl_sync(0xffffffffu, (unsigned long long)src, l);
      if (!m) return nullptr;
      m &= m - 1;
      return a;
    };
    for (int k = 0; k < G::NSK; ++k) {
      const int slot = G::SPLIT ? 0 : (sk + k) & 1;
      const char *a = take(issue);
      if (!a) break;
      if (G::SPLIT) {
        copy_part<G, 0>(ra, &bar[0], a, lane);
        copy_part<G, 1>(ra + G::KB, &bar[1], a, lane);
      } else {
        copy_part<G, 2>(ra + slot * G::SLOT, &bar[slot], a, lane);
      }
    }
    if (todo && !have_q) {  // under the first copies' latency
      load_q_tile(QuerySrc{p.q, b * p.q_sb + (int64_t)h * p.gqa * p.q_sh + i * p.q_sq, p.q_sh, p.q_dtype, p.gqa,
                           p.scale},
                  lane, f, qt);
      __syncwarp();
      have_q = true;
    }
    while (todo) {
      const int l = __ffs(todo) - 1;
      todo &= todo - 1;
      const int lo = __shfl_sync(0xffffffffu, vlo, l), hi = __shfl_sync(0xffffffffu, vhi, l);
      const char *next = take(issue);
      const bool ok = (lo == 0 && hi == G::C)
                          ? sparse_chunk<G, 0>(st, f, 0, G::C, region, bar, sk, ph, next, qa, qt, lane)
                          : sparse_chunk<G, 2>(st, f, lo, hi, region, bar, sk, ph, next, qa, qt, lane);
      if (!ok) {  // a copy never landed: record it, let what is in flight land (bounded), stop (results invalid)
        atomicExch(&g_sparse_fast_error, ERR_TIMEOUT_FULL);
        for (int k = 0; k < 2; ++k) ptx::mbar_wait_bounded(&bar[k], ph, WAIT_BUDGET);
        todo = 0;
        base = n;
      }
      if (++sk == G::NSK) {
        sk = 0;
        ph ^= 1u;
      }
    }
  }
  float *part = (float *)region;
  flush_to(p.gqa, st, part, part + 8, part + 16, lane);
}

template <class G>
__global__ void __launch_bounds__(kSW * 32, 2) sparse_kernel(const __grid_constant__ SparseParams p) {
  extern __shared__ __align__(128) unsigned char smem[];
  constexpr int kBars = kSW * 4 * 8, kWarpBytes = G::BUF + kQaBytes + kQTileBytes;
  static_assert(G::BUF >= kPartFloats * 4 && kWarpBytes % 16 == 0, "a partial lies in the copy buffers");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t *bar = (uint64_t *)smem + warp * 4;
  float *merged = (float *)(smem + kBars);  // this CTA's partial, for the cluster
  unsigned char *regions = smem + kBars + kPartFloats * 4;
  if (lane == 0) {
    for (int k = 0; k < 4; ++k) ptx::mbar_init(&bar[k], 1);
    ptx::fence_mbar_init();
  }
  __syncwarp();
  ptx::grid_dependency_wait();  // queries, lists, cache and length may come from the preceding kernel
  const int64_t T = sparse::launch_length(p.T, p.len_dev, p.q_len);
  if (T == 0 && blockIdx.x == 0 && threadIdx.x == 0) atomicExch(&g_sparse_fast_error, ERR_LENGTH);
  const int upc = kSW / p.w, gi = warp / p.w, rank = (int)(blockIdx.x % p.s);
  const unsigned unit = blockIdx.x / (unsigned)p.s * upc + gi;
  const bool live = unit < p.units;
  unsigned char *region = regions + warp * kWarpBytes;
  if (live && T > 0) {
    unit_main<G>(p, T, unit, rank * p.w + (warp - gi * p.w), region, bar, lane);
  } else {  // no length: an empty partial, so the rows come out as zeros
    float *part = (float *)region;
    if (lane < 8) part[lane] = -INFINITY, part[8 + lane] = 0.f;
    for (int k = lane; k < 8 * HD; k += 32) part[16 + k] = 0.f;
  }
  __syncthreads();
  // the group's w partials: weights 2^(m_w - M), four channels of a head per thread
  const int gt = p.w * 32, tid = threadIdx.x - gi * gt, Gq = p.gqa;
  const float *parts = (const float *)(regions + gi * p.w * kWarpBytes);
  constexpr int PS = kWarpBytes / 4;
  const unsigned bh = unit / (unsigned)p.q_len;  // output rows [b][h * Gq + g][i]: (bh * Gq + g) * q_len + i
  const int qi = (int)(unit - bh * (unsigned)p.q_len);
  auto finish = [&](int g, int d, float4 a, float M, float L) {
    const int64_t row = ((int64_t)bh * Gq + g) * p.q_len + qi;
    const float inv = L > 0.f ? 1.f / L : 0.f;
    store_from_float(p.out, row * HD + d, a.x * inv, p.out_dtype);
    store_from_float(p.out, row * HD + d + 1, a.y * inv, p.out_dtype);
    store_from_float(p.out, row * HD + d + 2, a.z * inv, p.out_dtype);
    store_from_float(p.out, row * HD + d + 3, a.w * inv, p.out_dtype);
    if (p.lse_out && d == 0) p.lse_out[row] = L > 0.f ? (M + log2f(L)) * LN2 : -INFINITY;
  };
  if (live) {
    for (int idx = tid; idx < Gq * (HD / 4); idx += gt) {
      const int g = idx / (HD / 4), d = (idx - g * (HD / 4)) * 4;
      float M = -INFINITY, L = 0.f;
      for (int k = 0; k < p.w; ++k) M = fmaxf(M, parts[k * PS + g]);
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int k = 0; k < p.w; ++k) {
        const float m = parts[k * PS + g];
        const float fk = m == -INFINITY ? 0.f : fast_exp2(m - M);
        const float4 o = *(const float4 *)(parts + k * PS + 16 + g * HD + d);
        L = fmaf(parts[k * PS + 8 + g], fk, L);
        a.x = fmaf(o.x, fk, a.x);
        a.y = fmaf(o.y, fk, a.y);
        a.z = fmaf(o.z, fk, a.z);
        a.w = fmaf(o.w, fk, a.w);
      }
      if (p.s == 1) {
        finish(g, d, a, M, L);
      } else {
        *(float4 *)(merged + 16 + g * HD + d) = a;
        if (d == 0) merged[g] = M, merged[8 + g] = L;
      }
    }
  }
  if (p.s == 1) return;
  // one unit per cluster: each CTA finishes its share of the rows from every CTA's partial
  cluster_sync();
  if (live) {
    const uint32_t mine = ptx::smem_u32(merged);
    for (int idx = rank + p.s * (int)threadIdx.x; idx < Gq * (HD / 4); idx += p.s * kSW * 32) {
      const int g = idx / (HD / 4), d = (idx - g * (HD / 4)) * 4;
      float m[kMaxCluster], l[kMaxCluster];
      float4 o[kMaxCluster];
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int c = 0; c < kMaxCluster; ++c) {
        if (c < p.s) {
          const uint32_t a = map_shared(mine, c);
          m[c] = ld_cluster(a + g * 4);
          l[c] = ld_cluster(a + (8 + g) * 4);
          o[c] = ld_cluster4(a + (16 + g * HD + d) * 4);
          M = fmaxf(M, m[c]);
        }
      }
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int c = 0; c < kMaxCluster; ++c) {
        if (c < p.s) {
          const float fk = m[c] == -INFINITY ? 0.f : fast_exp2(m[c] - M);
          L = fmaf(l[c], fk, L);
          a.x = fmaf(o[c].x, fk, a.x);
          a.y = fmaf(o[c].y, fk, a.y);
          a.z = fmaf(o[c].z, fk, a.z);
          a.w = fmaf(o[c].w, fk, a.w);
        }
      }
      finish(g, d, a, M, L);
    }
  }
  cluster_sync();  // no CTA leaves while another still reads its partial
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
struct SparseGeo : GeoSpec {
  void (*fn)(SparseParams);
  int smem;
};

template <int SK, int SV, int VP = 4>
static SparseGeo sparse_geo() {
  using G = Geo<SK, SV, VP>;
  return SparseGeo{geo_spec<G>(), sparse_kernel<G>,
                   kSW * 4 * 8 + kPartFloats * 4 + kSW * (G::BUF + kQaBytes + kQTileBytes)};
}

// The decode kernel's stride pairs and bit-plane formats.
static const SparseGeo *find_sparse_geo(int sk, int sv, int vp, int *index) {
  static const SparseGeo table[] = {
      sparse_geo<16, 8>(),     sparse_geo<16, 16>(),    sparse_geo<16, 32>(),    sparse_geo<16, 64>(),
      sparse_geo<32, 8>(),     sparse_geo<32, 16>(),    sparse_geo<32, 32>(),    sparse_geo<32, 64>(),
      sparse_geo<64, 8>(),     sparse_geo<64, 16>(),    sparse_geo<64, 32>(),    sparse_geo<64, 64>(),
      sparse_geo<64, 32, 3>(), sparse_geo<32, 8, 3>(), sparse_geo<64, 32, 2>(), sparse_geo<32, 8, 2>(),
  };
  for (int i = 0; i < (int)(sizeof(table) / sizeof(table[0])); ++i)
    if (table[i].sk == sk && table[i].sv == sv && table[i].vp == vp) {
      *index = i;
      return &table[i];
    }
  return nullptr;
}

static const SparseGeo *sparse_layout(const cq_paged_cache &c, int n_q_heads, int bt, int64_t *phs, int *index) {
  if (n_q_heads / c.kv_heads > 8 || !stored_for_mma(c)) return nullptr;
  const SparseGeo *g = find_sparse_geo(c.k.stride, c.v.stride, v_pack_of(c), index);
  if (!g || bt % g->C || !stored_as(c, *g, *phs)) return nullptr;
  return g;
}

// Warps per unit.  With W of them a unit takes about ceil(n / W) chunk times
// plus a fixed part of about 2.5 (lookups, query fragments, the merge); the
// machine runs 16 warps per SM at a time, and where that takes more than one
// round the last one is half empty.  The W with the least such time is taken.
// (4096 units of 32 chunks: 240, 217, 228, 256, 356 us with W = 1, 2, 4, 8, 16;
// 128 units of 64: 42, 25.6, 24.6, 31.9 us with 4, 8, 16, 32; 8 units of 64: 17.1,
// 12.1, 9.1, 7.8 us with 8, 16, 32, 64.)
static int pick_warps(int64_t units, int n, int sms) {
  const double slots = (double)sms * 2 * kSW;
  int best = 1;
  double best_t = 0;
  for (int W = 1; W <= kSW * kMaxCluster; W *= 2) {
    if (W > 1 && W > n) break;
    const double rounds = units * W / slots;
    const double t = (rounds <= 1 ? 1 : rounds + 0.5) * ((n + W - 1) / W + 2.5);
    if (W == 1 || t < best_t) {
      best = W;
      best_t = t;
    }
  }
  return best;
}

}  // namespace fast

bool sparse_fast_supported(const cq_paged_cache &c, int64_t T, int n_q_heads, int block_tokens) {
  int64_t phs;
  int index;
  return T + block_tokens < (1LL << 31) && fast::sparse_layout(c, n_q_heads, block_tokens, &phs, &index) != nullptr;
}

int run_sparse_fast(const cq_paged_cache &c, int64_t T, const int64_t *len_dev, const void *q, int q_dtype,
                    int n_q_heads, int q_len, int64_t q_sb, int64_t q_sh, int64_t q_sq, float scale,
                    const int64_t *starts, const int32_t *blocks, int top, int block_tokens, void *out, int out_dtype,
                    float *lse_out, cudaStream_t st) {
  using namespace fast;
  SparseParams p;
  int gi = 0;
  const SparseGeo *geo = sparse_layout(c, n_q_heads, block_tokens, &p.phs, &gi);
  CQ_REQUIRE(geo, CQ_ERR_UNSUPPORTED, "cq_sparse_attention: layout not taken");
  p.cv = make_view(c);
  p.blk = (const char *)c.k.keyframes;
  p.q = q;
  p.q_dtype = q_dtype;
  p.q_sb = q_sb;
  p.q_sh = q_sh;
  p.q_sq = q_sq;
  p.scale = scale;
  p.gqa = n_q_heads / c.kv_heads;
  p.q_len = q_len;
  p.top = top;
  p.bt = block_tokens;
  p.T = T;
  p.len_dev = len_dev;
  p.starts = starts;
  p.blocks = blocks;
  p.cpb = block_tokens / geo->C;
  p.units = (unsigned)((int64_t)c.batch * c.kv_heads * q_len);  // below 2^31 (the caller's check of the query rows)
  p.out = out;
  p.out_dtype = out_dtype;
  p.lse_out = lse_out;
  CQ_REQUIRE((int64_t)top * p.cpb < (1LL << 30), CQ_ERR_UNSUPPORTED, "cq_sparse_attention: list too long");
  const int W = pick_warps(p.units, top * p.cpb, sm_count());
  p.w = std::min(W, kSW);
  p.s = W / p.w;
  const int64_t grid = (p.units + kSW / p.w - 1) / (kSW / p.w) * p.s;
  CQ_REQUIRE(grid < (1LL << 31), CQ_ERR_INVALID, "cq_sparse_attention: grid too large");

  static std::mutex mu;
  static bool attr_set[64][32] = {};
  {
    int dev = 0;
    cudaGetDevice(&dev);
    std::lock_guard<std::mutex> lk(mu);
    if (dev < 0 || dev >= 64 || !attr_set[dev][gi]) {
      cudaError_t e = cudaFuncSetAttribute(geo->fn, cudaFuncAttributeMaxDynamicSharedMemorySize, geo->smem);
      if (e != cudaSuccess) {
        cudaGetLastError();
        return set_error(CQ_ERR_CUDA, std::string("cq_sparse_attention: ") + cudaGetErrorString(e));
      }
      if (dev >= 0 && dev < 64) attr_set[dev][gi] = true;
    }
  }
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)p.s;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kSW * 32);
  cfg.dynamicSmemBytes = (size_t)geo->smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaError_t e = cudaLaunchKernelEx(&cfg, geo->fn, p);
  if (e != cudaSuccess) {
    cudaGetLastError();  // reported here, not by the next call
    return set_error(CQ_ERR_CUDA, std::string("cq_sparse_attention: ") + cudaGetErrorString(e));
  }
  return check_launch("cq_sparse_attention");
}

int read_sparse_fast_error(int clear) {
  int v = 0;
  cudaMemcpyFromSymbol(&v, fast::g_sparse_fast_error, sizeof(int));
  if (clear && v) {
    const int z = 0;
    cudaMemcpyToSymbol(fast::g_sparse_fast_error, &z, sizeof(int));
  }
  return v;
}
int read_bounds_error_sparse_fast(int clear) { return read_bounds_error_here(clear); }

}  // namespace cq
