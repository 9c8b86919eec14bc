// Attention of one new token per request where groups of requests share the
// pages of a prefix (include/gguf_kv.h, gguf_kv_attn_shared).
//
// softmax(scale q . K) V over a prefix is a product of matrices: the rows of
// one side are the q heads of a kv head of all requests that share it.  A
// unit of work is such a block of rows against a stretch of positions: either
// rows of a group against the group's prefix, or the heads of one request
// against its own positions.  The tiles of all units form one line, which is
// cut evenly over the CTAs; every piece of a unit leaves the accumulators,
// maxima and sums of its rows, and sh_merge_kernel joins a request's pieces
// of both kinds.
#include <limits.h>
#include <math.h>

#include <cmath>

#include "paged_shared.cuh"

namespace vireo {

// ---- CUDA cores --------------------------------------------------------------
constexpr int kFmaThreads = 256;
template <int HS>
struct Fma {
  static constexpr int ROWS = HS == 256 ? 8 : 16, TILE = HS == 256 ? 32 : 64;  // of a unit, of a tile
  static constexpr int W = kFmaThreads / 32, PW = TILE / W, DQ = 32 / PW;  // positions of a warp at once, lanes to one
  static constexpr int KS = HS + DQ;  // of a row of keys: a quarter warp's reads fall into different banks
  static constexpr int RING = W * PW * (KS + HS), JOIN = W * ROWS * (HS + 2);
  static constexpr int SMEM = 4 * (ROWS * HS + RING + W * ROWS * (PW + 1));
  static_assert(JOIN <= RING, "the join takes the keys' and values' place");
};

// 16 bytes to shared memory, or the first `bytes` of them and zeros
VDEV void cp_async16_some(void* dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(bytes) : "memory");
}

// A unit of at most NR rows.  Each warp takes PW positions at a time for itself,
// with an online softmax of its own, and the warps join once, at the unit's end.
// While it works on the keys the values are on their way, and the other way
// round; no warp waits for another.  DQ lanes share a position's key, and a step's
// sums over them leave each lane NR / DQ rows.
//
// Two CTAs to an SM.  Up to eight rows of a prefix HBM and the start bound it (2
// groups of 6 x 16 heads behind 4097 positions: 38 us replayed, floor 18; one row, 8000
// positions: 43 us, 4.9 TB/s); from nine on reads of shared memory do, q's most
// (2 groups of 16: 64 us, of 32: 109).  Tiles shared by the CTA with barriers
// between loading, products and softmax took 60, 79 and 141; packed products with
// every weight held twice 40, 73 and 123.  16 rows of 256 dimensions do not fit the
// registers.
template <int HS, int NR>
VDEV void fma_unit(const ShParams& p, const ShUnit& w, float* sm) {
  using F = Fma<HS>;
  constexpr int PW = F::PW, DQ = F::DQ, NC = HS / (4 * DQ), RL = NR > DQ ? NR / DQ : 1, V = HS < 128 ? 2 : 4,
                NV = HS / (32 * V), PIECES = PW * HS / 128, STEP = F::W * PW;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, pos_l = lane % PW, dq = lane / PW;
  float* sq = sm;
  float* ring = sq + F::ROWS * HS;
  float *sk = ring + warp * PW * F::KS, *sv = ring + F::W * PW * F::KS + warp * PW * HS;
  float* sw = ring + F::RING + warp * F::ROWS * (PW + 1);  // [PW][NR] weights, then the rows' factors
  const int32_t* pages = w.pages(p);
  const int page = 1 << p.ps_shift;
  // without a sign: two steps behind the last position of the longest request
  const unsigned int len = w.len, end = min(len, (unsigned int)(w.tile + w.count) * F::TILE);
  const auto page_of = [&](unsigned int pos) { return pos < end ? pages[pos >> p.ps_shift] : 0; };
  const auto load = [&](const void* pool, float* dst, int stride, unsigned int pos, int id) {
    if (pos < end) {
      const bool there = id >= 0 && id < p.n_pages;
      if (!there) set_error(p.err, VIREO_ERR_ARG);
      const float* from = reinterpret_cast<const float*>(pool) + (there ? (int64_t)id * p.page_stride : 0) +
                          (int64_t)w.kh * p.head_stride;
#pragma unroll
      for (int i = 0; i < PIECES; i++) {
        const int x = lane + 32 * i, r = x / (HS / 4), c = x % (HS / 4) * 4;
        const bool has = there && pos + r < len;  // what is not there comes as zeros
        cp_async16_some(dst + r * stride + c, from + (has ? (int64_t)((pos + r) & (page - 1)) * p.pos_stride : 0) + c,
                        has ? 16 : 0);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  unsigned int pos = w.tile * F::TILE + warp * PW;
  int id = page_of(pos), next_id = page_of(pos + STEP);
  load(p.k, sk, F::KS, pos, id);
  load(p.v, sv, HS, pos, id);
  for (int x = tid; x < NR * (HS / 4); x += kFmaThreads) {
    const int r = x / (HS / 4), c = x % (HS / 4) * 4;
    float t[4] = {};
    if (r < w.rows) {
      int seq, head;
      w.row(p, r, seq, head);
      load_f<4>(reinterpret_cast<const float*>(p.q) + (int64_t)seq * p.q_stride + (int64_t)head * HS + c, t);
    }
    store_f<4>(sq + r * HS + c, t);
  }
  __syncthreads();
  int row0 = 0;  // this lane's rows
#pragma unroll
  for (int o = PW, n = NR; o < 32 && n > 1; o <<= 1, n /= 2) row0 += lane & o ? n / 2 : 0;
  float m[RL], l[RL], o[NR][NV][V] = {};
#pragma unroll
  for (int j = 0; j < RL; j++) {
    m[j] = -INFINITY;
    l[j] = 0.f;
  }
#pragma unroll 1
  for (; pos < end; pos += STEP) {
    const int ahead = page_of(pos + 2 * STEP);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
    float s[NR] = {};
#pragma unroll
    for (int i = 0; i < NC; i++) {
      const float4 k = *reinterpret_cast<const float4*>(sk + pos_l * F::KS + 4 * (dq + DQ * i));
#pragma unroll
      for (int r = 0; r < NR; r++) {
        const float4 x = *reinterpret_cast<const float4*>(sq + r * HS + 4 * (dq + DQ * i));
        s[r] += x.x * k.x;
        s[r] += x.y * k.y;
        s[r] += x.z * k.z;
        s[r] += x.w * k.w;
      }
    }
    __syncwarp();
    load(p.k, sk, F::KS, pos + STEP, next_id);
#pragma unroll
    for (int b = PW, n = NR; b < 32; b <<= 1, n = n > 1 ? n / 2 : 1) {
      if (n > 1) {
#pragma unroll
        for (int j = 0; j < n / 2; j++) {
          const float give = lane & b ? s[j] : s[j + n / 2], keep = lane & b ? s[j + n / 2] : s[j];
          s[j] = keep + __shfl_xor_sync(0xffffffffu, give, b);
        }
      } else {
        s[0] += __shfl_xor_sync(0xffffffffu, s[0], b);
      }
    }
    bool moved = false;
#pragma unroll
    for (int j = 0; j < RL; j++) {
      // rounded before the maximum is taken off: what a large product lost is no part of a weight
      const float x = pos + pos_l < len ? __fmul_rn(s[j], p.scale) : -INFINITY;
      float top = x;
#pragma unroll
      for (int b = 1; b < PW; b <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, b));
      top = fmaxf(top, m[j]);
      const float sub = top == -INFINITY ? 0.f : top;  // scores of -inf alone
      const float e = sh_ex2(x - sub), f = sh_ex2(m[j] - sub);
      moved |= top != m[j];
      m[j] = top;
      l[j] = l[j] * f + e;  // of this lane's position; over all at the end
      sw[pos_l * NR + row0 + j] = e;
      if (pos_l == 0) sw[PW * NR + row0 + j] = f;
    }
    moved = __any_sync(0xffffffffu, moved);  // and the weights are written
    __syncwarp();
    if (moved)
#pragma unroll
      for (int r = 0; r < NR; r++) {
        const float f = sw[PW * NR + r];
#pragma unroll
        for (int d = 0; d < NV; d++)
#pragma unroll
          for (int e = 0; e < V; e++) o[r][d][e] *= f;
      }
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
#pragma unroll
    for (int j = 0; j < PW; j++) {
      float e[NR];
      if constexpr (NR % 4 == 0) {
#pragma unroll
        for (int r = 0; r < NR; r += 4) {
          const float4 x = *reinterpret_cast<const float4*>(sw + j * NR + r);
          e[r] = x.x;
          e[r + 1] = x.y;
          e[r + 2] = x.z;
          e[r + 3] = x.w;
        }
      } else {
#pragma unroll
        for (int r = 0; r < NR; r++) e[r] = sw[j * NR + r];
      }
#pragma unroll
      for (int d = 0; d < NV; d++) {
        float x[V];
        load_f<V>(sv + j * HS + V * (lane + 32 * d), x);
#pragma unroll
        for (int r = 0; r < NR; r++)
#pragma unroll
          for (int c = 0; c < V; c++) o[r][d][c] += e[r] * x[c];
      }
    }
    __syncwarp();
    load(p.v, sv, HS, pos + STEP, next_id);
    next_id = ahead;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();  // keys and values are read: their place for the join
  float *jm = ring + F::W * F::ROWS * HS, *jl = jm + F::W * F::ROWS;
#pragma unroll
  for (int j = 0; j < RL; j++) {
#pragma unroll
    for (int b = 1; b < PW; b <<= 1) l[j] += __shfl_xor_sync(0xffffffffu, l[j], b);
    if (pos_l == 0) {
      jm[warp * F::ROWS + row0 + j] = m[j];
      jl[warp * F::ROWS + row0 + j] = l[j];
    }
  }
#pragma unroll
  for (int r = 0; r < NR; r++)
#pragma unroll
    for (int d = 0; d < NV; d++) store_f<V>(ring + (warp * F::ROWS + r) * HS + V * (lane + 32 * d), o[r][d]);
  __syncthreads();
  for (int x = tid; x < w.rows * (HS / 4); x += kFmaThreads) {
    const int r = x / (HS / 4), c = x % (HS / 4) * 4;
    float top = -INFINITY, sum = 0.f, acc[4] = {};
#pragma unroll
    for (int v = 0; v < F::W; v++) top = fmaxf(top, jm[v * F::ROWS + r]);
    const float sub = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int v = 0; v < F::W; v++) {
      const float f = sh_ex2(jm[v * F::ROWS + r] - sub);
      const float4 y = *reinterpret_cast<const float4*>(ring + (v * F::ROWS + r) * HS + c);
      sum += jl[v * F::ROWS + r] * f;
      acc[0] += y.x * f;
      acc[1] += y.y * f;
      acc[2] += y.z * f;
      acc[3] += y.w * f;
    }
    float* st = p.part + (int64_t)(w.part + r) * (HS + 4);
    store_f<4>(st + c, acc);
    if (c == 0) {
      st[HS] = top;
      st[HS + 1] = sum;
    }
  }
}

template <int HS>
__global__ void __launch_bounds__(kFmaThreads, 2) sh_fma_kernel(const __grid_constant__ ShParams p) {
  extern __shared__ __align__(16) float sm[];
  pdl_launch_dependents();
  pdl_wait();
  const ShStretch my = sh_plan<kFmaThreads, false>(p, reinterpret_cast<uint8_t*>(sm));
#pragma unroll 1
  for (int u = 0; u < my.n; u++) {
    const ShUnit w = my.units[u];
    __syncthreads();  // the last one's join is done
    if (w.rows == 1)
      fma_unit<HS, 1>(p, w, sm);
    else if (w.rows <= 4)
      fma_unit<HS, 4>(p, w, sm);
    else if (w.rows <= 8)
      fma_unit<HS, 8>(p, w, sm);
    else if constexpr (HS < 256)
      fma_unit<HS, 16>(p, w, sm);
  }
}

// ---- join ----------------------------------------------------------------------
// A warp per (request, head), or a CTA where those are few.  The maxima and sums
// of up to 32 pieces are read at once, a lane each, and give every piece its
// factor; then the accumulators are added, several on their way at a time.  With
// WARPS on one row, each takes every WARPS-th piece and the first joins them.
constexpr int kShMergeWarps = 4;
template <class TA, int HS, int WARPS>
__global__ void __launch_bounds__(32 * kShMergeWarps) sh_merge_kernel(const __grid_constant__ ShParams p) {
  constexpr int V = HS / 32 < 4 ? 2 : 4, NV = HS / (32 * V), ROW = HS + 4;
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, part = warp % WARPS;
  const unsigned int item = blockIdx.x * (kShMergeWarps / WARPS) + warp / WARPS;
  if (item >= (unsigned int)(p.n_seqs * p.H)) return;  // one row to a CTA: all of it or nothing
  const int lane = threadIdx.x & 31, i = (int)(item / (unsigned int)p.H), head = (int)item - i * p.H;
  const int kh = (int)((unsigned int)head / (unsigned int)p.R), hr = head - kh * p.R;
  const ShReq q = p.all[i];
  const ShReq a = p.all[max(q.lead, 0)];
  const int total = *p.total;
  const ShCut cut(max(total, 1), total ? sh_ctas(p, total) : 1);
  const int nto = sh_tiles(p, q.own);
  const int own = q.line + (q.prefix ? p.G * sh_blocks(p, q.members) * sh_tiles(p, q.prefix) : 0) +
                  (kh * p.nsub + (hr >> p.rt_shift)) * nto;
  // pieces of the request's own positions, and of its group's prefix: rows of the first CTA's, and CTAs
  int c0 = 0, n0 = 0, c1 = 0, n1 = 0;
  int64_t row0 = 0, row1 = 0;
  if (nto > 0) {
    c0 = cut.of(own);
    n0 = cut.of(own + nto - 1) - c0 + 1;
    row0 = (int64_t)q.row0 + (q.prefix ? q.members * p.H : 0) + head + (int64_t)p.rt * c0;
  }
  if (q.lead >= 0) {
    const int f = (i - q.lead) * p.R + hr, nt = sh_tiles(p, a.prefix);
    const int line = a.line + (kh * sh_blocks(p, a.members) + (f >> p.rt_shift)) * nt;
    c1 = cut.of(line);
    n1 = cut.of(line + nt - 1) - c1 + 1;
    row1 = (int64_t)a.row0 + kh * a.members * p.R + f + (int64_t)p.rt * c1;
  }
  const int n = (n0 + n1 - part + WARPS - 1) / WARPS;
  float m = -INFINITY, l = 0.f, o[NV][V] = {};
  for (int base = 0; base < n; base += 32) {
    const int j = (base + lane) * WARPS + part;
    const float* st = p.part + (j < n0 ? row0 + (int64_t)p.rt * j : row1 + (int64_t)p.rt * (j - n0)) * ROW;
    float mm = -INFINITY, ll = 0.f;
    if (base + lane < n) {
      mm = st[HS];
      ll = st[HS + 1];
    }
    float mn = fmaxf(m, mm);
#pragma unroll
    for (int d = 16; d; d >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, d));
    const float sub = mn == -INFINITY ? 0.f : mn, f = sh_ex2(m - sub), g = sh_ex2(mm - sub);
    ll *= g;
#pragma unroll
    for (int d = 16; d; d >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, d);
    l = l * f + ll;
    m = mn;
#pragma unroll
    for (int d = 0; d < NV; d++)
#pragma unroll
      for (int e = 0; e < V; e++) o[d][e] *= f;
    const int here = min(32, n - base);
    const int64_t at = st - p.part;
#pragma unroll 4
    for (int x = 0; x < here; x++) {
      const float* from = p.part + __shfl_sync(0xffffffffu, at, x);
      const float w = __shfl_sync(0xffffffffu, g, x);
#pragma unroll
      for (int d = 0; d < NV; d++) {
        float v[V];
        load_f<V>(from + V * (lane + 32 * d), v);
#pragma unroll
        for (int e = 0; e < V; e++) o[d][e] += v[e] * w;
      }
    }
  }
  if constexpr (WARPS > 1) {
    __shared__ float so[WARPS][HS], sm[WARPS], sl[WARPS];
    if (part) {
#pragma unroll
      for (int d = 0; d < NV; d++) store_f<V>(&so[part][V * (lane + 32 * d)], o[d]);
      if (lane == 0) {
        sm[part] = m;
        sl[part] = l;
      }
    }
    __syncthreads();
    if (part) return;
    float mn = m;
#pragma unroll
    for (int w = 1; w < WARPS; w++) mn = fmaxf(mn, sm[w]);
    const float sub = mn == -INFINITY ? 0.f : mn, f = sh_ex2(m - sub);
    l *= f;
#pragma unroll
    for (int d = 0; d < NV; d++)
#pragma unroll
      for (int e = 0; e < V; e++) o[d][e] *= f;
#pragma unroll
    for (int w = 1; w < WARPS; w++) {
      const float g = sh_ex2(sm[w] - sub);
      l += sl[w] * g;
#pragma unroll
      for (int d = 0; d < NV; d++) {
        float v[V];
        load_f<V>(&so[w][V * (lane + 32 * d)], v);
#pragma unroll
        for (int e = 0; e < V; e++) o[d][e] += v[e] * g;
      }
    }
  }
  const float f = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);  // a NaN stays one
#pragma unroll
  for (int d = 0; d < NV; d++) {
#pragma unroll
    for (int e = 0; e < V; e++) o[d][e] *= f;
    store_f<V>(reinterpret_cast<TA*>(p.out) + (int64_t)i * p.out_stride + (int64_t)head * HS + V * (lane + 32 * d), o[d]);
  }
}

// ---- host ------------------------------------------------------------------------
template <class TA, int HS>
static const void* sh_merge_w(bool few) {
  return few ? reinterpret_cast<const void*>(&sh_merge_kernel<TA, HS, kShMergeWarps>)
             : reinterpret_cast<const void*>(&sh_merge_kernel<TA, HS, 1>);
}
template <class TA>
static const void* sh_merge_h(int hs, bool few) {
  return hs == 64 ? sh_merge_w<TA, 64>(few) : hs == 128 ? sh_merge_w<TA, 128>(few) : sh_merge_w<TA, 256>(few);
}
static const void* sh_merge(const gguf_kv_desc& d, bool few) {
  return d.act_type == KV_BF16  ? sh_merge_h<__nv_bfloat16>(d.head_size, few)
         : d.act_type == KV_F16 ? sh_merge_h<__half>(d.head_size, few)
                                : sh_merge_h<float>(d.head_size, few);
}
template <int HS>
static ShKernel sh_fma() {
  return {reinterpret_cast<const void*>(&sh_fma_kernel<HS>), kFmaThreads, Fma<HS>::SMEM, Fma<HS>::ROWS, Fma<HS>::TILE,
          false, 0, 2};
}
static ShKernel sh_kernel_for(const gguf_kv_desc& d) {
  if (d.kv_type == KV_F32) return d.head_size == 64 ? sh_fma<64>() : d.head_size == 128 ? sh_fma<128>() : sh_fma<256>();
  return sh_mma_kernel(d);
}

static size_t sh_up(size_t v) { return (v + 255) & ~(size_t)255; }
struct ShWs {
  size_t units, all, total, part, img, up, eights, bytes;
};
static ShWs sh_ws(const gguf_kv_desc& d, int n_seqs) {
  const ShKernel k = sh_kernel_for(d);
  const int nsub = (d.n_heads / d.n_kv_heads + k.rt - 1) / k.rt;
  // of a request's own, and of the prefix of a group, which has no more blocks of rows than its members together
  const size_t ctas = (size_t)kShaSms * k.per_sm, units = 2 * (size_t)n_seqs * d.n_kv_heads * nsub + ctas;
  const size_t rows = 2 * (size_t)n_seqs * d.n_heads + ctas * k.rt,
               eights = k.img ? 2 * (size_t)n_seqs * d.n_kv_heads * ((d.n_heads / d.n_kv_heads + 7) / 8) + 16 * ctas : 0;
  ShWs w;
  w.units = 0;
  w.all = sh_up(units * sizeof(ShUnit));
  w.total = w.all + sh_up((size_t)n_seqs * sizeof(ShReq));
  w.part = w.total + 256;
  w.img = w.part + sh_up(rows * (d.head_size + 4) * 4);
  w.up = w.img + sh_up(eights * k.img);
  w.eights = w.up + sh_up(eights * 8);
  w.bytes = w.eights + sh_up(eights * sizeof(ShEight));
  return w;
}
// Rows of an SM up to which a CTA takes one: as many CTAs as it holds at once.  256
// rows of 37 pieces and more: 81.6 us for the call (replayed), a warp each 93.2; 2048 rows
// of ten 45.7 and 45.8; 64 rows of two 16.5 and 16.4.
constexpr int kShMergeFew = 16;
constexpr int kShaRows = 1 << 20;  // q heads of all requests
static bool sh_shape(const gguf_kv_desc& d, int n_seqs, int n_groups) {
  return n_seqs <= kShaSeqs && n_groups <= kShaSeqs && (int64_t)n_seqs * d.n_heads <= kShaRows &&
         d.n_heads / d.n_kv_heads <= 128;
}

}  // namespace vireo

using namespace vireo;

extern "C" {

size_t gguf_kv_shared_workspace(const gguf_kv* kv, int n_seqs, int n_groups) {
  if (!kv || n_seqs < 0 || n_groups < 0 || !sh_shape(kv->d, n_seqs, n_groups)) return 0;
  return sh_ws(kv->d, n_seqs).bytes;
}

int gguf_kv_attn_shared(gguf_kv* kv, const gguf_kv_attn_args* a, const gguf_kv_group_args* g, void* stream) {
  int st = kv_attn_check(kv, a);
  if (st) return st;
  if (!g || g->n_groups < 0) return VIREO_ERR_ARG;
  const gguf_kv_desc& d = kv->d;
  if (!sh_shape(d, a->n_seqs, g->n_groups)) return VIREO_ERR_UNSUPPORTED;
  if (a->n_seqs == 0) return VIREO_OK;
  if (!g->cu || (g->n_groups > 0 && !g->shared) || a->ws_bytes < sh_ws(d, a->n_seqs).bytes)
    return VIREO_ERR_ARG;
  const ShKernel k = sh_kernel_for(d);
  // tiles of all requests as long as the table is wide, each twice: of a prefix and of its own
  const int64_t nsub = (d.n_heads / d.n_kv_heads + k.rt - 1) / k.rt;
  if ((((int64_t)a->max_pages * d.page_size + k.tile - 1) / k.tile + 1) * d.n_kv_heads * nsub >
      INT32_MAX / 2 / a->n_seqs)
    return VIREO_ERR_UNSUPPORTED;
  Ctx* c = ctx_get(&st);
  if (!c) return st;
  DeviceGuard dg(c->device);
  if (dg.status) return dg.status;
  const ShWs w = sh_ws(d, a->n_seqs);
  uint8_t* ws = (uint8_t*)a->ws;
  ShParams p;
  p.q = a->q;
  p.k = d.k;
  p.v = d.v;
  p.out = a->out;
  p.q_stride = a->q_stride;
  p.out_stride = a->out_stride;
  p.table_stride = a->table_stride;
  p.page_stride = d.page_stride;
  p.head_stride = d.head_stride;
  p.pos_stride = d.pos_stride;
  p.table = a->table;
  p.kv_len = a->kv_len;
  p.cu = g->cu;
  p.shared = g->shared;
  p.n_seqs = a->n_seqs;
  p.max_pages = a->max_pages;
  p.n_pages = d.n_pages;
  p.n_groups = g->n_groups;
  p.H = d.n_heads;
  p.G = d.n_kv_heads;
  p.R = d.n_heads / d.n_kv_heads;
  p.ps_shift = kv->ps_shift;
  p.rt = k.rt;
  p.nsub = (p.R + k.rt - 1) / k.rt;
  p.rt_shift = p.tile_shift = 0;
  while ((1 << p.rt_shift) < k.rt) p.rt_shift++;
  while ((1 << p.tile_shift) < k.tile) p.tile_shift++;
  p.ctas = std::min(kShaSms, c->num_sms) * k.per_sm;
  p.scale = (a->scale == 0.f ? 1.0f / sqrtf((float)d.head_size) : a->scale) * kShaLog2e;
  p.units = (ShUnit*)(ws + w.units);
  p.all = (ShReq*)(ws + w.all);
  p.total = (int*)(ws + w.total);
  p.part = (float*)(ws + w.part);
  p.img = ws + w.img;
  p.up = (int8_t*)(ws + w.up);
  p.eights = (ShEight*)(ws + w.eights);
  p.err = c->d_err;
  cudaStream_t s = stream ? (cudaStream_t)stream : c->stream;
  const int smem = std::max(k.smem, (int)sh_plan_smem(a->n_seqs, g->n_groups));
  // the most of any call: another thread's may come between this and the launch
  if ((st = cuda_status(cudaFuncSetAttribute(k.fn, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             std::max(k.smem, (int)sh_plan_smem(kShaSeqs, kShaSeqs))))))
    return st;
  CUtensorMap mk, mv;
  if (k.maps) {
    std::lock_guard<std::mutex> lk(kv->mu);
    if (!kv->wide_ok) {
      if ((st = kv_make_map(d, k.tile, &kv->wide_k, d.k)) || (st = kv_make_map(d, k.tile, &kv->wide_v, d.v))) return st;
      kv->wide_ok = true;
    }
    mk = kv->wide_k;
    mv = kv->wide_v;
  }
  void* args[] = {&p, &mk, &mv};
  if ((st = launch_pdl_c(k.fn, dim3(p.ctas), dim3(k.threads), smem, s, args))) return st;
  const int rows = a->n_seqs * p.H;
  const bool few = rows <= kShMergeFew * c->num_sms;
  return launch_pdl_c(sh_merge(d, few), dim3(few ? rows : (rows + kShMergeWarps - 1) / kShMergeWarps),
                      dim3(32 * kShMergeWarps), 0, s, args);
}

}  // extern "C"
