// The paged key-value pool (include/gguf_kv.h): the handle, block tables and
// slot maps from request lengths, and the append of new tokens (bias, QK
// norm, rotation, cache write, page means).  The attention over the pool is
// in paged_attn.cu.
#include <math.h>
#include <string.h>

#include <new>

#include "gguf_compute.h"
#include "paged_kv.cuh"
#include "pdl_launch.cuh"

namespace vireo {

// ---------------------------------------------------------------------------
// Block tables and slot maps.
//
// Everything follows from four prefix sums over the requests (new pages and
// tokens asked for; tokens granted; pages given back), integers throughout.
// One cluster of CTAs: each CTA computes all of the prefix sums for itself
// (a few thousand lengths, in shared memory afterwards), the per-token work
// is then spread over the cluster's threads.  A token finds its request by
// binary search in the granted prefix sums, and its page in the table (pages
// that were there) or in the ring (new ones: the j-th new page of a call is
// ring[head + j], known without communication).  The cluster barrier between
// reading the lengths and the state and writing them lets a caller update
// both in place.  Latency-bound: the whole call moves a few bytes per token.
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;
constexpr int kPlanMaxSeqs = 8192;
constexpr int kPlanMaxCtas = 8;

struct PlanParams {
  gguf_kv_plan_args a;
  int ps_shift;
};

// inclusive prefix sums over the block of three values per thread; returns
// the block totals in tot
struct Plan3 {
  long long need, ask, back;
};
VDEV Plan3 add3(const Plan3& x, const Plan3& y) { return {x.need + y.need, x.ask + y.ask, x.back + y.back}; }

VDEV Plan3 block_scan3(Plan3 v, Plan3* red, Plan3& tot) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    Plan3 u;
    u.need = __shfl_up_sync(0xffffffffu, v.need, o);
    u.ask = __shfl_up_sync(0xffffffffu, v.ask, o);
    u.back = __shfl_up_sync(0xffffffffu, v.back, o);
    if (lane >= o) v = add3(v, u);
  }
  __syncthreads();  // red may still be read from the previous scan
  if (lane == 31) red[warp] = v;
  __syncthreads();
  Plan3 before = {0, 0, 0};
  tot = before;
  for (int w = 0; w < nw; w++) {
    if (w < warp) before = add3(before, red[w]);
    tot = add3(tot, red[w]);
  }
  return add3(v, before);
}

__global__ void __launch_bounds__(kPlanThreads) kv_plan_kernel(const __grid_constant__ PlanParams p) {
  pdl_wait();
  extern __shared__ int sh[];
  const gguf_kv_plan_args& a = p.a;
  const int n = a.n_seqs, tid = threadIdx.x, nt = blockDim.x;
  int* cu = sh;            // [n + 1] granted tokens before each request
  int* past = cu + n + 1;  // [n]
  int* rank = past + n;    // [n] new pages before each request; of an end, pages given back before it
  __shared__ Plan3 red[kPlanThreads / 32];
  const int page = 1 << p.ps_shift;
  const unsigned int np = (unsigned int)a.n_pages;
  const unsigned int head = (unsigned int)a.state[0] % np;
  const long long count = min(max(a.state[1], 0), a.n_pages);
  const unsigned int rank_in = blockIdx.x, nblk = gridDim.x;  // one cluster is the whole grid

  Plan3 carry = {0, 0, 0};
  long long cu_carry = 0, taken = 0;
  for (int base = 0; base < n; base += nt) {
    const int i = base + tid;
    int pa = 0, ad = 0, ok = 0;
    Plan3 v = {0, 0, 0};
    if (i < n) {
      pa = a.past[i];
      ad = a.add[i];
      const long long want = ((long long)pa + max(ad, 0) + page - 1) >> p.ps_shift;
      ok = pa >= 0 && ad >= -1 && want <= a.max_pages;
      if (ok) {
        const long long have = ((long long)pa + page - 1) >> p.ps_shift;
        v.need = want - have;
        v.ask = max(ad, 0);
        v.back = ad < 0 ? have : 0;
      }
    }
    Plan3 tot;
    const Plan3 upto = add3(block_scan3(v, red, tot), carry);
    const int granted =
        ok && (v.need == 0 || upto.need <= count) && (v.ask == 0 || upto.ask <= (long long)a.n_slots);
    Plan3 g = {granted ? v.need : 0, granted ? v.ask : 0, 0}, gtot;
    const Plan3 gu = block_scan3(g, red, gtot);
    if (i < n) {
      cu[i] = (int)(cu_carry + gu.ask - g.ask);
      past[i] = pa;
      rank[i] = (int)(ad < 0 ? upto.back - v.back : upto.need - v.need);
      if (!granted) rank[i] = -1;
    }
    cu_carry += gtot.ask;
    taken += gtot.need;
    carry = add3(carry, tot);
  }
  if (tid == 0) cu[n] = (int)cu_carry;
  // every CTA of the cluster has read past, add and state before any of
  // them is written in place
  asm volatile("barrier.cluster.arrive.aligned;\n barrier.cluster.wait.aligned;" ::: "memory");
  const int total = (int)cu_carry;
  // tokens
  const int gt = rank_in * nt + tid, gn = nblk * nt;
  for (int t = gt; t < a.n_slots; t += gn) {
    int64_t slot = -1;
    int pos = 0;
    if (t < total) {
      int lo = 0, hi = n;  // the last request with cu[i] <= t holds the token
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid] <= t) lo = mid;
        else hi = mid;
      }
      pos = past[lo] + (t - cu[lo]);
      const int have = (int)(((long long)past[lo] + page - 1) >> p.ps_shift), pi = pos >> p.ps_shift;
      int32_t* row = a.table + (int64_t)lo * a.table_stride;
      int id;
      if (pi < have) {
        id = row[pi];
      } else {
        id = a.ring[(head + (unsigned int)(rank[lo] + pi - have)) % np];
        if ((pos & (page - 1)) == 0) row[pi] = id;  // a page's first token enters it in the table
      }
      slot = ((int64_t)id << p.ps_shift) + (pos & (page - 1));
    }
    a.slots[t] = slot;
    a.pos[t] = pos;
  }
  // requests
  for (int i = gt; i <= n; i += gn) {
    a.cu[i] = cu[i];
    if (i < n) {
      const int add = a.add[i], ok = rank[i] >= 0, got = cu[i + 1] - cu[i];
      a.granted[i] = ok;
      a.kv_len[i] = ok && add < 0 ? 0 : max(past[i] + got, 0);
    }
  }
  // pages of ended requests, a warp to a request, behind the ring's last free one
  const int warp = gt >> 5, lane = tid & 31, nwarp = gn >> 5;
  for (int i = warp; i < n; i += nwarp) {
    if (rank[i] < 0 || a.add[i] >= 0) continue;
    const int have = (int)(((long long)past[i] + page - 1) >> p.ps_shift);
    const int32_t* row = a.table + (int64_t)i * a.table_stride;
    for (int j = lane; j < have; j += 32)
      a.ring[(head + (unsigned long long)count + (unsigned int)rank[i] + j) % np] = row[j];
  }
  if (gt == 0) {
    a.state_out[0] = (int)((head + (unsigned long long)taken) % np);
    a.state_out[1] = (int)(count - taken + carry.back);
  }
}

// ---------------------------------------------------------------------------
// Append: a row (one head of one token) is held by LPR = HS / E neighbouring
// lanes, E values each, loaded and stored 16 bytes at a time; its sum of
// squares is a shuffle reduction over the lanes, and the partner of a
// rotated value sits LPR-internally in another lane at the same register, so
// one pass over the data does bias, norm, rotation and the cache write with
// nothing staged.  The cosines and sines of a token's position are formed
// once per CTA (64-bit revolutions, reduced, then fp32) and shared by all
// its heads.  A CTA takes `tpb` tokens and the rows [y * rpc, ...) of each; a
// full-width norm sums the token's whole row again in every CTA that needs it
// (it is in L2 by then).  Memory-bound.
// ---------------------------------------------------------------------------
constexpr int kAppThreads = 256;
constexpr int kAppMaxTpb = 4;

struct AppendParams {
  gguf_kv_append_args a;
  void *kc, *vc;
  int64_t page_stride, head_stride, pos_stride;
  int H, G, ps_shift, rope, tpb, rpc;
  int64_t n_slots;
  float eps;
  int* err;
  KvFreq f;
};

template <int LPR>
VDEV float row_sum(float v) {
#pragma unroll
  for (int o = LPR / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <class TA, class TC, int HS>
__global__ void __launch_bounds__(kAppThreads) kv_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int E = 16 / (int)sizeof(TA) > HS / 32 ? 16 / (int)sizeof(TA) : HS / 32;
  constexpr int LPR = HS / E, RPW = 32 / LPR, NW = kAppThreads / 32;
  __shared__ float2 cs[kAppMaxTpb][kKvMaxHalf];
  __shared__ float ss[kAppMaxTpb][2];
  __shared__ int64_t slot_s[kAppMaxTpb];
  pdl_launch_dependents();
  pdl_wait();
  const gguf_kv_append_args& a = p.a;
  const int t0 = blockIdx.x * p.tpb, ntok = min(p.tpb, a.n_tokens - t0);
  const int rows = p.H + 2 * p.G, r0 = blockIdx.y * p.rpc, nrow = min(p.rpc, rows - r0);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, half = p.rope >> 1;
  if (tid < ntok) {
    int64_t s = a.slots[t0 + tid];
    if (s >= p.n_slots) {
      set_error(p.err, VIREO_ERR_ARG);
      s = -1;
    }
    slot_s[tid] = s;
  }
  for (int i = tid; i < ntok * half; i += kAppThreads) {
    const int t = i / half, j = i - t * half;
    const double rev = (double)a.pos[t0 + t] * p.f.rev[j];
    float c, s;
    sincospif(2.0f * (float)(rev - rint(rev)), &s, &c);
    cs[t][j] = make_float2(c, s);
  }
  // full-width norms: the whole row's sum of squares, a warp to a (token, q or k)
  const bool qfull = a.q_norm && a.q_norm_len != HS, kfull = a.k_norm && a.k_norm_len != HS;
  if (qfull || kfull)
    for (int job = warp; job < 2 * ntok; job += NW) {
      const int t = job >> 1, isk = job & 1, w = (isk ? p.G : p.H) * HS;
      if (isk ? !kfull || r0 + nrow <= p.H || r0 >= p.H + p.G : !qfull || r0 >= p.H) continue;
      const TA* x = isk ? (const TA*)a.k + (int64_t)(t0 + t) * a.k_stride : (const TA*)a.q + (int64_t)(t0 + t) * a.q_stride;
      const float* b = isk ? a.bk : a.bq;
      float s = 0.f;
      for (int i = lane * E; i < w; i += 32 * E) {
        float v[E];
        load_f<E>(x + i, v);
#pragma unroll
        for (int e = 0; e < E; e++) {
          if (b) v[e] += b[i + e];
          s += v[e] * v[e];
        }
      }
      s = row_sum<32>(s);
      if (lane == 0) ss[t][isk] = s;
    }
  __syncthreads();
  const int sub = lane / LPR, l = lane % LPR, n = ntok * nrow;
  for (int it = warp * RPW; it < n; it += NW * RPW) {
    // a lane group past the end repeats the last row's loads (its lanes take
    // part in the shuffles) and stores nothing
    const int idx = min(it + sub, n - 1);
    const int t = idx / nrow, r = r0 + idx - t * nrow;
    const int64_t slot = slot_s[t];
    const bool live = it + sub < n && slot >= 0;
    const int kind = r < p.H ? 0 : r < p.H + p.G ? 1 : 2, h = kind == 0 ? r : kind == 1 ? r - p.H : r - p.H - p.G;
    const int64_t tok = t0 + t;
    const TA* src = (kind == 0 ? (const TA*)a.q + tok * a.q_stride
                               : kind == 1 ? (const TA*)a.k + tok * a.k_stride : (const TA*)a.v + tok * a.v_stride) +
                    h * HS + l * E;
    float v[E];
    load_f<E>(src, v);
    const float* b = kind == 0 ? a.bq : kind == 1 ? a.bk : a.bv;
    if (b) {
      float u[E];
      load_f<E>(b + h * HS + l * E, u);
#pragma unroll
      for (int e = 0; e < E; e++) v[e] += u[e];
    }
    const float* nw = kind == 0 ? a.q_norm : kind == 1 ? a.k_norm : nullptr;
    float sq = 0.f;
#pragma unroll
    for (int e = 0; e < E; e++) sq += v[e] * v[e];
    sq = row_sum<LPR>(sq);  // every lane takes part, whatever its row's kind
    if (nw) {
      const bool full = kind == 0 ? qfull : kfull;
      const float s = full ? ss[t][kind] : sq;
      const int len = full ? (kind == 0 ? p.H : p.G) * HS : HS;
      const float rs = 1.0f / sqrtf(s / (float)len + p.eps);
      float u[E];
      load_f<E>(nw + (full ? h * HS : 0) + l * E, u);
#pragma unroll
      for (int e = 0; e < E; e++) v[e] = v[e] * rs * u[e];
    }
    if (half) {  // the partner of dimension j is j +- half; half is a multiple of E
      const int hl = half / E;
      const bool turned = kind < 2 && l < 2 * hl, upper = l >= hl;
      const int other = turned ? (upper ? lane - hl : lane + hl) : lane;
      const int j0 = (upper ? l - hl : l) * E;
#pragma unroll
      for (int e = 0; e < E; e++) {
        const float w = __shfl_sync(0xffffffffu, v[e], other);
        if (turned) {
          const float2 c = cs[t][j0 + e];
          v[e] = upper ? w * c.y + v[e] * c.x : v[e] * c.x - w * c.y;
        }
      }
    }
    if (!live) continue;
    if (kind == 0) {
      store_f<E>((TA*)a.q_out + tok * a.q_out_stride + h * HS + l * E, v);
    } else {
      TC* c = (TC*)(kind == 1 ? p.kc : p.vc) + (slot >> p.ps_shift) * p.page_stride + (int64_t)h * p.head_stride +
              (slot & ((1 << p.ps_shift) - 1)) * p.pos_stride + l * E;
      store_f<E>(c, v);
    }
  }
}

// Means of the pages whose last position the append wrote: a CTA looks at 32
// tokens' slots; for each that ends a page its warps take the kv heads in
// turn, a lane group per position, and sum the page's keys in fp32.
constexpr int kMeanTok = 32;
template <class TC, int HS>
__global__ void __launch_bounds__(256) kv_means_kernel(const __grid_constant__ AppendParams p) {
  constexpr int E = 16 / (int)sizeof(TC) > HS / 32 ? 16 / (int)sizeof(TC) : HS / 32;
  constexpr int LPR = HS / E, RPW = 32 / LPR;
  pdl_launch_dependents();
  pdl_wait();
  const int page = 1 << p.ps_shift, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = blockIdx.x * kMeanTok + lane;
  int64_t s = t < p.a.n_tokens ? p.a.slots[t] : -1;
  const bool ends = s >= 0 && s < p.n_slots && (int)(s & (page - 1)) == page - 1;
  unsigned int todo = __ballot_sync(0xffffffffu, ends);  // the same in every warp of the CTA
  const int npg = __popc(todo);
  for (int job = warp; job < npg * p.G; job += 8) {
    const int which = job / p.G, g = job - which * p.G;
    unsigned int m = todo;
    for (int i = 0; i < which; i++) m &= m - 1;
    const int64_t pg = __shfl_sync(0xffffffffu, s, __ffs(m) - 1) >> p.ps_shift;
    const int sub = lane / LPR, l = lane % LPR;
    const TC* k = (const TC*)p.kc + pg * p.page_stride + (int64_t)g * p.head_stride + l * E;
    float acc[E];
#pragma unroll
    for (int e = 0; e < E; e++) acc[e] = 0.f;
#pragma unroll 8
    for (int o = sub; o < page; o += RPW) {  // page >= 8 >= RPW, a multiple of it
      float v[E];
      load_f<E>(k + (int64_t)o * p.pos_stride, v);
#pragma unroll
      for (int e = 0; e < E; e++) acc[e] += v[e];
    }
#pragma unroll
    for (int e = 0; e < E; e++) {
#pragma unroll
      for (int o = LPR; o < 32; o <<= 1) acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], o);
      acc[e] *= 1.0f / (float)page;  // exact: a power of two
    }
    if (sub == 0) store_f<E>((TC*)p.a.means + (pg * p.G + g) * HS + l * E, acc);
  }
}

template <class TA, class TC, int HS>
static int launch_append(const AppendParams& p, dim3 grid, cudaStream_t s) {
  int st = pdl_launch(kv_append_kernel<TA, TC, HS>, grid, dim3(kAppThreads), 0, s, p);
  if (!st && p.a.means)
    st = pdl_launch(kv_means_kernel<TC, HS>, dim3((p.a.n_tokens + kMeanTok - 1) / kMeanTok), dim3(256), 0, s, p);
  return st;
}
template <class TA, class TC>
static int launch_append_h(const AppendParams& p, int hs, dim3 grid, cudaStream_t s) {
  switch (hs) {
    case 64: return launch_append<TA, TC, 64>(p, grid, s);
    case 128: return launch_append<TA, TC, 128>(p, grid, s);
    default: return launch_append<TA, TC, 256>(p, grid, s);
  }
}

}  // namespace vireo

using namespace vireo;

extern "C" {

int gguf_kv_create(const gguf_kv_desc* desc, gguf_kv** out) {
  if (!desc || !out) return VIREO_ERR_ARG;
  *out = nullptr;
  const gguf_kv_desc& d = *desc;
  if (d.n_heads < 1 || d.n_kv_heads < 1 || d.n_heads % d.n_kv_heads || d.n_heads > 65535 || d.head_size < 1 ||
      d.page_size < 1 || d.n_pages < 1 || !d.k || !d.v || !(d.eps >= 0.f) || !(d.rope_base > 0.f) ||
      d.rope_dim < 0 || d.rope_dim > d.head_size)
    return VIREO_ERR_ARG;
  if (!kv_aligned(d.k, 16) || !kv_aligned(d.v, 16)) return VIREO_ERR_ARG;
  const bool types = (d.act_type == KV_F32 && (d.kv_type == KV_F32 || d.kv_type == KV_F16)) ||
                     (d.act_type == d.kv_type && (d.kv_type == KV_F16 || d.kv_type == KV_BF16));
  if (!types || (d.head_size != 64 && d.head_size != 128 && d.head_size != 256) || d.page_size < 8 ||
      d.page_size > 1024 || (d.page_size & (d.page_size - 1)) || d.rope_dim % 16)
    return VIREO_ERR_UNSUPPORTED;
  const int el = kv_type_size(d.kv_type);
  // strides in whole 16 bytes, below the 2^40 bytes a tensor map takes
  const int64_t extent[3] = {d.n_pages, d.n_kv_heads, d.page_size};
  int64_t stride[3] = {d.page_stride, d.head_stride, d.pos_stride};
  for (int i = 0; i < 3; i++) {
    if (extent[i] == 1) stride[i] = d.head_size;
    if (stride[i] < d.head_size || stride[i] >= (1ll << 40) / el || (stride[i] * el) % 16) return VIREO_ERR_ARG;
  }
  gguf_kv* kv = new (std::nothrow) gguf_kv;
  if (!kv) return VIREO_ERR_NOMEM;
  kv->d = d;
  kv->d.page_stride = stride[0];
  kv->d.head_stride = stride[1];
  kv->d.pos_stride = stride[2];
  kv->ps_shift = 0;
  while ((1 << kv->ps_shift) < d.page_size) kv->ps_shift++;
  const double twopi = 6.283185307179586476925286766559;
  for (int j = 0; j < kKvMaxHalf; j++)
    kv->freq.rev[j] = j < d.rope_dim / 2 ? pow((double)d.rope_base, -2.0 * j / d.rope_dim) / twopi : 0.0;
  *out = kv;
  return VIREO_OK;
}

void gguf_kv_destroy(gguf_kv* kv) { delete kv; }

int gguf_kv_sync(gguf_kv* kv, void* stream) {
  if (!kv) return VIREO_ERR_ARG;
  return vireo_sync(stream);
}

int gguf_kv_plan(const gguf_kv_plan_args* a, void* stream) {
  if (!a || a->n_seqs < 0 || a->n_slots < 0 || a->n_pages < 1 || a->max_pages < 1 || a->page_size < 1 ||
      a->table_stride < a->max_pages || !a->ring || !a->state || !a->cu || !a->state_out ||
      (a->n_seqs > 0 && (!a->past || !a->add || !a->table || !a->kv_len || !a->granted)) ||
      (a->n_slots > 0 && (!a->slots || !a->pos)) || (int64_t)a->max_pages * a->page_size > INT32_MAX)
    return VIREO_ERR_ARG;
  if (a->n_seqs > kPlanMaxSeqs || a->page_size < 8 || a->page_size > 1024 || (a->page_size & (a->page_size - 1)))
    return VIREO_ERR_UNSUPPORTED;
  int st;
  Ctx* c = ctx_get(&st);
  if (!c) return st;
  DeviceGuard dg(c->device);
  if (dg.status) return dg.status;
  PlanParams p;
  p.a = *a;
  p.ps_shift = 0;
  while ((1 << p.ps_shift) < a->page_size) p.ps_shift++;
  // a thread per request or token up to one CTA, then as many CTAs as give
  // one, up to the portable cluster size
  const int items = std::max(a->n_seqs, a->n_slots);
  const int ctas = std::min(kPlanMaxCtas, std::max(1, (items + kPlanThreads - 1) / kPlanThreads));
  const int threads = std::min(kPlanThreads, std::max(64, (items + 31) / 32 * 32));
  const size_t smem = (size_t)(3 * a->n_seqs + 1) * sizeof(int);
  if (smem > 48 * 1024 &&
      (st = cuda_status(cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)((3 * kPlanMaxSeqs + 1) * sizeof(int))))))
    return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream ? (cudaStream_t)stream : c->stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cuda_status(cudaLaunchKernelEx(&cfg, kv_plan_kernel, p));
}

int gguf_kv_append(gguf_kv* kv, const gguf_kv_append_args* a, void* stream) {
  if (!kv || !a || a->n_tokens < 0) return VIREO_ERR_ARG;
  const gguf_kv_desc& d = kv->d;
  const int el = kv_type_size(d.act_type), hs = d.head_size;
  const int64_t qw = (int64_t)d.n_heads * hs, kw = (int64_t)d.n_kv_heads * hs;
  if ((a->q_norm && a->q_norm_len != hs && a->q_norm_len != qw) ||
      (a->k_norm && a->k_norm_len != hs && a->k_norm_len != kw))
    return VIREO_ERR_ARG;
  if (a->n_tokens == 0) return VIREO_OK;
  for (const void* ptr : {a->q, a->k, a->v, (const void*)a->q_out})
    if (!ptr || !kv_aligned(ptr, 16)) return VIREO_ERR_ARG;
  if (!a->pos || !a->slots || !kv_stride_ok(a->q_stride, qw, el) || !kv_stride_ok(a->k_stride, kw, el) ||
      !kv_stride_ok(a->v_stride, kw, el) || !kv_stride_ok(a->q_out_stride, qw, el) || !kv_aligned(a->means, 16))
    return VIREO_ERR_ARG;
  for (const void* ptr : {a->bq, a->bk, a->bv, a->q_norm, a->k_norm})
    if (!kv_aligned(ptr, 16)) return VIREO_ERR_ARG;
  int st;
  Ctx* c = ctx_get(&st);
  if (!c) return st;
  DeviceGuard dg(c->device);
  if (dg.status) return dg.status;
  AppendParams p;
  p.a = *a;
  p.kc = d.k;
  p.vc = d.v;
  p.page_stride = d.page_stride;
  p.head_stride = d.head_stride;
  p.pos_stride = d.pos_stride;
  p.H = d.n_heads;
  p.G = d.n_kv_heads;
  p.ps_shift = kv->ps_shift;
  p.rope = d.rope_dim;
  p.n_slots = (int64_t)d.n_pages * d.page_size;
  p.eps = d.eps;
  p.err = c->d_err;
  p.f = kv->freq;
  const int rows = d.n_heads + 2 * d.n_kv_heads;
  p.tpb = 1;
  p.rpc = rows;
  const dim3 grid((a->n_tokens + p.tpb - 1) / p.tpb, (rows + p.rpc - 1) / p.rpc);
  cudaStream_t s = stream ? (cudaStream_t)stream : c->stream;
  if (d.act_type == KV_BF16) return launch_append_h<__nv_bfloat16, __nv_bfloat16>(p, hs, grid, s);
  if (d.act_type == KV_F16) return launch_append_h<__half, __half>(p, hs, grid, s);
  if (d.kv_type == KV_F16) return launch_append_h<float, __half>(p, hs, grid, s);
  return launch_append_h<float, float>(p, hs, grid, s);
}

}  // extern "C"
