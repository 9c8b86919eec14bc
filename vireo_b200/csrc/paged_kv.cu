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
// Everything follows from prefix sums over the requests (new pages and tokens
// asked for, pages given back; tokens granted), integers throughout.  Each
// CTA computes all of them for itself (a few thousand lengths, in shared
// memory afterwards), and the tokens are spread over the grid's threads.  A
// token finds its request by binary search in the granted prefix sums, and
// its page in the table (pages that were there) or in the ring (new ones:
// the j-th new page of a call is ring[head + j], known without
// communication).  Where the lengths or the state are updated in place the
// grid is one cluster, whose barrier stands between reading and writing
// them; for more tokens than a cluster's threads a second launch of one
// computes and writes those alone.  Latency-bound: a call moves a few bytes
// per token (512 requests, 66k tokens, replayed: 6.1 us, with four tokens to
// a thread and a quarter of the CTAs 7.6).
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 512;
constexpr int kPlanMaxSeqs = 8192;
constexpr int kPlanMaxCluster = 8;
constexpr int kPlanMaxSlots = 1 << 30;

enum PlanPart { kPlanAll, kPlanTokens, kPlanLengths };  // kPlanLengths: kv_len and state_out; kPlanTokens: the rest
struct PlanParams {
  gguf_kv_plan_args a;
  int ps_shift;
  PlanPart part;
};

struct Plan3 {
  unsigned int need, ask, back;
};
// Sums that stop at 2^31 - 1: associative, and no length wraps them.  That is
// above any n_slots, and where a sum of pages stops there the tokens that ask
// for them, never fewer, do too, so nobody who asks is granted on it.
VDEV unsigned int add_cap(unsigned int x, unsigned int y) { return min(x + y, (unsigned int)INT32_MAX); }
VDEV Plan3 add3(const Plan3& x, const Plan3& y) {
  return {add_cap(x.need, y.need), add_cap(x.ask, y.ask), add_cap(x.back, y.back)};
}

VDEV Plan3 shfl3(const Plan3& v, int lane) {
  return {__shfl_sync(0xffffffffu, v.need, lane), __shfl_sync(0xffffffffu, v.ask, lane),
          __shfl_sync(0xffffffffu, v.back, lane)};
}
// inclusive prefix sums over a warp's first N lanes
template <int N>
VDEV Plan3 warp_scan3(Plan3 v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < N; o <<= 1) {
    const Plan3 u = {__shfl_up_sync(0xffffffffu, v.need, o), __shfl_up_sync(0xffffffffu, v.ask, o),
                     __shfl_up_sync(0xffffffffu, v.back, o)};
    if (lane >= o) v = add3(v, u);
  }
  return v;
}
// inclusive prefix sums over the block; tot: the block's
VDEV Plan3 block_scan3(Plan3 v, Plan3* red, Plan3& tot) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  v = warp_scan3<32>(v);
  __syncthreads();  // red may still be read from the previous scan
  if (lane == 31) red[warp] = v;
  __syncthreads();
  const Plan3 x = warp_scan3<kPlanThreads / 32>(lane < nw ? red[lane] : Plan3{0, 0, 0});
  tot = shfl3(x, nw - 1);
  const Plan3 before = shfl3(x, max(warp - 1, 0));
  return warp ? add3(v, before) : v;
}

__global__ void __launch_bounds__(kPlanThreads) kv_plan_kernel(const __grid_constant__ PlanParams p) {
  pdl_launch_dependents();
  pdl_wait();
  extern __shared__ int sh[];
  const gguf_kv_plan_args& a = p.a;
  const int n = a.n_seqs, tid = threadIdx.x, nt = blockDim.x;
  int* cu = sh;            // [n + 1] granted tokens before each request
  int* past = cu + n + 1;  // [n]
  int* rank = past + n;    // [n] new pages before each request; refused: -1; an end: -2 - pages given back before it
  __shared__ Plan3 red[kPlanThreads / 32];
  const int page = 1 << p.ps_shift;
  const unsigned int np = (unsigned int)a.n_pages;
  const unsigned int head0 = (unsigned int)a.state[0];
  const int count = min(max(a.state[1], 0), a.n_pages);

  Plan3 carry = {0, 0, 0};
  int cu_carry = 0, taken = 0;  // of what is granted: at most n_slots and count
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
        const int have = (int)(((long long)pa + page - 1) >> p.ps_shift);
        v.need = (unsigned int)((int)want - have);
        v.ask = (unsigned int)max(ad, 0);
        v.back = ad < 0 ? (unsigned int)have : 0u;
      }
    }
    Plan3 tot;
    const Plan3 upto = add3(block_scan3(v, red, tot), carry);
    const int granted = ok && (v.need == 0 || upto.need <= (unsigned int)count) &&
                        (v.ask == 0 || upto.ask <= (unsigned int)a.n_slots);
    Plan3 g = {granted ? v.need : 0u, granted ? v.ask : 0u, 0u}, gtot = tot;
    unsigned int before = upto.ask - carry.ask - v.ask;  // within this block of requests, all granted
    if (__syncthreads_or((v.need | v.ask) && !granted)) before = block_scan3(g, red, gtot).ask - g.ask;
    if (i < n) {
      cu[i] = cu_carry + (int)before;
      past[i] = pa;
      // pages given back before this end: no more than the ring has, where the state is right
      const int given = (int)min(upto.back - v.back, (unsigned int)INT32_MAX - 1u);
      rank[i] = !granted ? -1 : ad < 0 ? -2 - given : (int)(upto.need - v.need);
    }
    cu_carry += (int)gtot.ask;
    taken += (int)gtot.need;
    carry = add3(carry, tot);
  }
  if (tid == 0) cu[n] = cu_carry;
  const unsigned int head = head0 % np;
  // shared sums are complete; and every CTA of a cluster has read past, add
  // and state before any of them is written in place
  asm volatile("barrier.cluster.arrive.aligned;\n barrier.cluster.wait.aligned;" ::: "memory");
  const int total = cu_carry;
  const int gt = blockIdx.x * nt + tid, gn = gridDim.x * nt;
  const bool lengths = p.part != kPlanTokens;
  if (p.part != kPlanLengths) {
    for (int t = gt; t < a.n_slots; t += gn) {
      int64_t slot = -1;
      int pos = 0;
      if (t < total) {
        int i = 0;  // the last request with cu[i] <= t holds the token
        for (int step = 1 << (31 - __clz(n)); step; step >>= 1)
          if (i + step < n && cu[i + step] <= t) i += step;
        pos = past[i] + (t - cu[i]);
        const int have = (int)(((long long)past[i] + page - 1) >> p.ps_shift), pi = pos >> p.ps_shift;
        int32_t* entry = a.table + (int64_t)i * a.table_stride + pi;
        const int off = pos & (page - 1);
        const int id = pi < have ? *entry : a.ring[(head + (unsigned int)(rank[i] + pi - have)) % np];
        if (off == 0 && pi >= have) *entry = id;  // a new page's first token
        slot = ((int64_t)id << p.ps_shift) + off;
      }
      a.slots[t] = slot;
      a.pos[t] = pos;
    }
    // pages of ended requests, a warp to a request, behind the ring's last free one
    const int warp = gt >> 5, lane = tid & 31, nwarp = gn >> 5;
    for (int i = warp; i < n; i += nwarp) {
      if (rank[i] >= -1) continue;
      const int have = (int)(((long long)past[i] + page - 1) >> p.ps_shift);
      const int32_t* row = a.table + (int64_t)i * a.table_stride;
#pragma unroll 4
      for (int j = lane; j < have; j += 32)
        a.ring[(head + (unsigned long long)count + (unsigned int)(-2 - rank[i]) + j) % np] = row[j];
    }
  }
  // requests
  for (int i = gt; i <= n; i += gn) {
    if (p.part != kPlanLengths) a.cu[i] = cu[i];
    if (i < n) {
      if (p.part != kPlanLengths) a.granted[i] = rank[i] != -1;
      if (lengths) a.kv_len[i] = rank[i] < -1 ? 0 : max(past[i] + cu[i + 1] - cu[i], 0);
    }
  }
  if (lengths && gt == 0) {
    a.state_out[0] = (int)((head + (unsigned long long)taken) % np);
    a.state_out[1] = (int)min((long long)count - taken + carry.back, (long long)INT32_MAX);
  }
}

// ---------------------------------------------------------------------------
// Append: a row (one head of one token) is held by HS / 8 neighbouring lanes
// as eight values each, four of the first and the four that the rotation
// pairs them with of the second half, so that bias, norm, rotation and cache
// write need no exchange but the norm's sum (a shuffle reduction over the
// lanes) and one pass over the data does it all with nothing staged.  A lane
// group takes `rpg` rows of one token: its cosines and sines (64-bit
// revolutions, reduced, then fp32), with the per-head norm weights folded in,
// stay in registers for all of them.  Rows come through a ring in shared
// memory that asynchronous copies keep full, every thread copying what it
// reads itself, so that no barrier is needed; loads into registers, four rows
// at a time, left half the bytes in flight (8192 tokens of 40 rows of 128 bf16
// values, 168 MB: 45 us against 34).  With a full-width norm the groups of a
// CTA share one token and first sum its whole row together; its rows are then
// read again, from L2 (1368 tokens of 160 rows of 256 fp32 values: 233 us with
// the whole row summed in every group that needs it).
// Multiplies and adds are fused where written so, and nowhere else: a row's
// bits depend neither on its place in the group nor on the number of tokens.
// Bound by HBM and, nearly as much, by the number of instructions: hence the
// packed fp32 pairs.
// ---------------------------------------------------------------------------
constexpr int kAppThreads = 256;
constexpr int kAppAheadBytes = 64;  // of the rows ahead, per thread
constexpr int kAppFill = 4;         // CTAs per SM that the rows are spread over

struct AppendParams {
  gguf_kv_append_args a;
  void *kc, *vc;
  int64_t page_stride, head_stride, pos_stride;
  int H, G, ps_shift, rope;
  int rpg, groups;  // rows per lane group; lane groups per token, or CTAs with a full-width norm
  int team, stages;  // kv_append_team_kernel: warps to a token, a power of two; tokens in its ring
  int64_t n_slots;
  float eps, per_q, per_k;  // 1 / the full widths
  int* err;
  KvFreq f;
};

// four values as loaded
template <class T>
struct Raw4 {
  uint32_t w[sizeof(T)];
  VDEV void load(const T* p) {
    if constexpr (sizeof(T) == 4)
      *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p);
    else
      *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
  }
  VDEV void get(f2* o) const {
    const T* t = reinterpret_cast<const T*>(w);
    o[0] = f2_make(to_f(t[0]), to_f(t[1]));
    o[1] = f2_make(to_f(t[2]), to_f(t[3]));
  }
};
// the thread's own copies into its ring
VDEV void cp_async8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
VDEV void cp_async16_at(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
VDEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
VDEV void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
template <class T>
VDEV void store4(T* p, const f2* v) {
  float t[4];
  f2_get(v[0], t[0], t[1]);
  f2_get(v[1], t[2], t[3]);
  store_f<4>(p, t);
}

template <int LPR>
VDEV float row_sum(float v, unsigned mask) {
#pragma unroll
  for (int o = LPR / 2; o; o >>= 1) v += __shfl_xor_sync(mask, v, o);
  return v;
}

// a lane's eight of a row of fp32 values (biases, weights)
VDEV void load8(const float* p, int o1, int o2, f2 (&u)[4]) {
  load4(p + o1, u);
  load4(p + o2, u + 2);
}
VDEV void add8(const f2 (&u)[4], f2 (&y)[4]) {
#pragma unroll
  for (int e = 0; e < 4; e++) y[e] = f2_add(y[e], u[e]);
}
VDEV void mul8(const f2 (&u)[4], f2 (&y)[4]) {
#pragma unroll
  for (int e = 0; e < 4; e++) y[e] = f2_mul(y[e], u[e]);
}
// a row's sum of squares, in all its lanes
template <int LPR>
VDEV float row_sumsq(const f2 (&y)[4], unsigned mask) {
  f2 sq = f2_mul(y[0], y[0]);
#pragma unroll
  for (int e = 1; e < 4; e++) sq = f2_fma(y[e], y[e], sq);
  float s0, s1;
  f2_get(sq, s0, s1);
  return row_sum<LPR>(s0 + s1, mask);
}

// The sum of squares of a full width.  Head i's goes to part[i mod
// kAppParts], and those are added in an order that the number of heads alone
// decides: how rows are spread over threads does not change a bit.
constexpr int kAppParts = 256;
VDEV void put_part(float* part, int i, float x) {
  part[i & (kAppParts - 1)] = i < kAppParts ? x : part[i & (kAppParts - 1)] + x;
}
VDEV float sum_parts(const float* part, int n) {  // by a whole warp
  float x = 0.f;
  for (int i = threadIdx.x & 31; i < min(n, kAppParts); i += 32) x += part[i];
  return row_sum<32>(x, 0xffffffffu);
}

// A lane's part of the rotation with the per-head norm weights (or ones)
// folded in: y1' = a1 y1 + b2 y2, y2' = b1 y1 + a2 y2 (a = c w, b = -+ s w).
struct Turn {
  f2 a1[2], a2[2], b1[2], b2[2];
  VDEV void set(const float (&c)[4], const float (&s)[4], const float* w, int o1, int o2) {
    f2 w1[2] = {f2_make(1.f, 1.f), f2_make(1.f, 1.f)}, w2[2] = {w1[0], w1[1]};
    if (w) {
      load4(w + o1, w1);
      load4(w + o2, w2);
    }
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const f2 ce = f2_make(c[2 * e], c[2 * e + 1]);
      a1[e] = f2_mul(ce, w1[e]);
      a2[e] = f2_mul(ce, w2[e]);
      b1[e] = f2_mul(f2_make(s[2 * e], s[2 * e + 1]), w1[e]);
      b2[e] = f2_mul(f2_make(-s[2 * e], -s[2 * e + 1]), w2[e]);
    }
  }
  VDEV void apply(float f, const f2 (&y)[4], f2 (&z)[4]) const {
    const f2 ff = f2_make(f, f);
#pragma unroll
    for (int e = 0; e < 2; e++) {
      z[e] = f2_mul(ff, f2_fma(b2[e], y[2 + e], f2_mul(a1[e], y[e])));
      z[2 + e] = f2_mul(ff, f2_fma(b1[e], y[e], f2_mul(a2[e], y[2 + e])));
    }
  }
};
// cosine and sine of a position's angle: revolutions reduced in 64 bits
VDEV float2 app_angle(int pos, double per_pos) {
  const double rev = (double)pos * per_pos;
  float sn, cn;
  sincospif(2.0f * (float)(rev - rint(rev)), &sn, &cn);
  return make_float2(cn, sn);
}

// What a call needs besides per-head norms: their loads and branches are not
// in the loop of the calls without.
enum AppendMode { kAppPlain, kAppBias, kAppFull };  // kAppFull: a full-width norm, and perhaps biases
template <class TA, class TC, int HS, int MODE>
__global__ void __launch_bounds__(kAppThreads, MODE ? 3 : 4) kv_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr bool GEN = MODE != kAppPlain;
  constexpr int LPR = HS / 8, GPB = kAppThreads / LPR, PART = 4 * (int)sizeof(TA), AHEAD = kAppAheadBytes / (2 * PART);
  __shared__ __align__(16) uint8_t ring[AHEAD][kAppThreads * 2 * PART];
  pdl_launch_dependents();
  pdl_wait();
  const gguf_kv_append_args& a = p.a;
  const int lane = threadIdx.x & 31, l = lane % LPR;
  const unsigned mask = LPR == 32 ? 0xffffffffu : ((1u << LPR) - 1u) << (lane / LPR * LPR);
  const int grp = threadIdx.x / LPR, rows = p.H + 2 * p.G;
  int64_t tok;
  int rg;
  if constexpr (MODE == kAppFull) {
    tok = blockIdx.x / p.groups;
    rg = (int)(blockIdx.x - tok * p.groups) * GPB + grp;
  } else {  // neighbouring groups take neighbouring tokens' same rows
    const int64_t item = (int64_t)blockIdx.x * GPB + grp;
    if (item >= (int64_t)a.n_tokens * p.groups) return;
    rg = (int)(item / a.n_tokens);
    tok = item - (int64_t)rg * a.n_tokens;
  }
  const int64_t slot = a.slots[tok];
  const int pos = a.pos[tok];
  const int r0 = min(rows, rg * p.rpg), r1 = min(rows, r0 + p.rpg);
  // a skipped token's rows are read like any other's and not written, so that
  // no load waits for the slot
  const bool live = slot >= 0 && slot < p.n_slots;
  if (slot >= p.n_slots && l == 0) set_error(p.err, VIREO_ERR_ARG);
  const int64_t at =
      live ? (slot >> p.ps_shift) * p.page_stride + (slot & ((1 << p.ps_shift) - 1)) * p.pos_stride : 0;
  // this lane's dimensions: o1 .. o1 + 3 and o2 .. o2 + 3, pairs of the
  // rotation below rope / 2 (a multiple of 8) and of nothing behind it
  const int half = p.rope >> 1, rest = (HS - p.rope) >> 1, j0 = 4 * l;
  const bool turned = j0 < half;
  const int o1 = turned ? j0 : p.rope + (j0 - half), o2 = o1 + (turned ? half : rest);
  const TA *q = (const TA*)a.q + tok * a.q_stride, *k = (const TA*)a.k + tok * a.k_stride,
           *v = (const TA*)a.v + tok * a.v_stride;
  // one group of copies per row, empty behind the last: row r is there when
  // all but the latest AHEAD - 1 groups are.  16-bit: both parts in 16 bytes;
  // fp32: 16 bytes each, apart by the block's, so that a warp's reads of
  // either meet no bank conflict.
  constexpr int SIDE = PART == 16 ? kAppThreads * 16 : 8;
  const uint32_t mine = smem_addr(&ring[0][0]) + threadIdx.x * 16;
  const auto issue = [&](int r) {
    if (r < r1) {
      const TA* x = r < p.H ? q + r * HS : r < p.H + p.G ? k + (r - p.H) * HS : v + (r - p.H - p.G) * HS;
      const uint32_t dst = mine + (uint32_t)(r & (AHEAD - 1)) * sizeof(ring[0]);
      if constexpr (PART == 16) {
        cp_async16_at(dst, x + o1);
        cp_async16_at(dst + SIDE, x + o2);
      } else {
        cp_async8(dst, x + o1);
        cp_async8(dst + SIDE, x + o2);
      }
    }
    cp_async_commit();
  };
  const auto fetch = [&](int r, f2 (&y)[4]) {
    cp_async_wait<AHEAD - 1>();
    const uint8_t* src = &ring[r & (AHEAD - 1)][threadIdx.x * 16];
    Raw4<TA> r1_, r2_;
    if constexpr (PART == 16) {
      r1_.load(reinterpret_cast<const TA*>(src));
      r2_.load(reinterpret_cast<const TA*>(src + SIDE));
    } else {
      const uint4 w = *reinterpret_cast<const uint4*>(src);
      r1_.w[0] = w.x;
      r1_.w[1] = w.y;
      r2_.w[0] = w.z;
      r2_.w[1] = w.w;
    }
    r1_.get(y);
    r2_.get(y + 2);
    issue(r + AHEAD);
  };
#pragma unroll
  for (int i = 0; i < AHEAD; i++) issue(r0 + i);
  float c[4] = {1.f, 1.f, 1.f, 1.f}, s[4] = {0.f, 0.f, 0.f, 0.f};
  if (MODE != kAppFull && turned && r0 < p.H + p.G)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float2 cs = app_angle(pos, p.f.rev[j0 + e]);
      c[e] = cs.x;
      s[e] = cs.y;
    }

  // Full-width factors: every CTA of a token sums all of its heads.
  float fq = 1.f, fk = 1.f;
  if constexpr (MODE == kAppFull) {
    __shared__ float part[2][kAppParts];
    __shared__ float2 turns[kKvMaxHalf];  // the token's angles, once
    if ((int)threadIdx.x < half) turns[threadIdx.x] = app_angle(pos, p.f.rev[threadIdx.x]);
    const int c0 = (rg - grp) * p.rpg, c1 = c0 + GPB * p.rpg;  // this CTA's rows of the token
    const bool nq = a.q_norm && a.q_norm_len != HS && c0 < p.H;
    const bool nk = a.k_norm && a.k_norm_len != HS && c1 > p.H && c0 < p.H + p.G;
    const auto sums = [&](const TA* x, const float* b, int n, float* to) {
#pragma unroll 4
      for (int i = grp; i < n; i += GPB) {
        Raw4<TA> r1_, r2_;
        r1_.load(x + i * HS + o1);
        r2_.load(x + i * HS + o2);
        f2 y[4];
        r1_.get(y);
        r2_.get(y + 2);
        if (b) {
          f2 u[4];
          load8(b + i * HS, o1, o2, u);
          add8(u, y);
        }
        const float sq = row_sumsq<LPR>(y, mask);
        if (l == 0) put_part(to, i, sq);
      }
    };
    if (nq) sums(q, a.bq, p.H, part[0]);
    if (nk) sums(k, a.bk, p.G, part[1]);
    __syncthreads();  // and no row is replaced in place before all are summed
    if (turned)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        c[e] = turns[j0 + e].x;
        s[e] = turns[j0 + e].y;
      }
    if (nq) fq = rsqrtf(fmaf(sum_parts(part[0], p.H), p.per_q, p.eps));
    if (nk) fk = rsqrtf(fmaf(sum_parts(part[1], p.G), p.per_k, p.eps));
  }

  // q and k rows [h0, h1); full: the factor of a full-width norm
  const auto turn = [&](const float* bias, const float* nw, int norm_len, float full_f, int first, int h0, int h1,
                        auto&& put) {
    if (h0 >= h1) return;
    const bool full = MODE == kAppFull && nw && norm_len != HS;
    Turn t;
    t.set(c, s, full ? nullptr : nw, o1, o2);
    float f = full ? full_f : 1.f;
    // a row's biases are loaded a row ahead, weights before the wait for its
    // copy (8192 tokens, 16 / 16 heads of 128, bf16, per-head norms and biases:
    // 53 us against 62 with loads behind the wait)
    f2 ub[4];
    if (GEN && bias) load8(bias + h0 * HS, o1, o2, ub);
#pragma unroll 2
    for (int h = h0; h < h1; h++) {
      f2 y[4], z[4], uw[4];
      if (full) load8(nw + h * HS, o1, o2, uw);
      fetch(first + h, y);
      if (GEN && bias) {
        add8(ub, y);
        if (h + 1 < h1) load8(bias + (h + 1) * HS, o1, o2, ub);
      }
      if (full)
        mul8(uw, y);
      else if (nw)
        f = rsqrtf(fmaf(row_sumsq<LPR>(y, mask), 1.0f / HS, p.eps));
      t.apply(f, y, z);
      put(h, z);
    }
  };
  TA* qo = (TA*)a.q_out + tok * a.q_out_stride;
  turn(a.bq, a.q_norm, a.q_norm_len, fq, 0, r0, min(r1, p.H), [&](int h, const f2* z) {
    if (!live) return;
    store4(qo + h * HS + o1, z);
    store4(qo + h * HS + o2, z + 2);
  });
  TC* ko = (TC*)p.kc + at;
  turn(a.bk, a.k_norm, a.k_norm_len, fk, p.H, max(r0 - p.H, 0), min(r1 - p.H, p.G), [&](int h, const f2* z) {
    if (!live) return;
    store4(ko + h * p.head_stride + o1, z);
    store4(ko + h * p.head_stride + o2, z + 2);
  });
  TC* vo = (TC*)p.vc + at;
  for (int h = max(r0 - p.H - p.G, 0); h < r1 - p.H - p.G; h++) {
    f2 y[4], u[4];
    if (GEN && a.bv) load8(a.bv + h * HS, o1, o2, u);
    fetch(p.H + p.G + h, y);
    if (GEN && a.bv) add8(u, y);
    if (!live) continue;
    store4(vo + h * p.head_stride + o1, y);
    store4(vo + h * p.head_stride + o2, y + 2);
  }
}

// Full-width norms of many tokens.  A CTA per token spends most of its time
// waiting (slot, rows, angles, the sum's barrier, then the rows), so here a
// team of warps takes one token after another: its rows are on their way to
// shared memory (every thread copying what it reads, twice) while the
// `stages` - 1 tokens before it are worked on, and a token costs one barrier
// of the team.  The smaller the team, the fewer instructions a token costs.
// Heads are dealt out to the team's lane groups, q, k and v apart.  Sums and
// angles alternate between two buffers, so that a warp that is ahead writes
// the one that nobody reads.  Bound by neither HBM (25 % of it) nor issue
// slots (45 %): 16 warps to an SM wait in turn for copies, weights and the
// steps of a sum (8192 tokens, 16 / 16 heads of 128: bf16 70 us, f32 / f16 75;
// a CTA per token 108 and 121; 32 warps of 64 registers were slower).
constexpr int kTeamThreads = 256, kTeamCtas = 2;  // per SM
template <class TA, class TC, int HS>
__global__ void __launch_bounds__(kTeamThreads, kTeamCtas)
    kv_append_team_kernel(const __grid_constant__ AppendParams p) {
  constexpr int LPR = HS / 8, RPW = 32 / LPR, PART = 4 * (int)sizeof(TA), COL = 2 * PART * kTeamThreads;
  extern __shared__ __align__(16) uint8_t shared[];
  pdl_launch_dependents();
  const gguf_kv_append_args& a = p.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % LPR;
  const unsigned mask = LPR == 32 ? 0xffffffffu : ((1u << LPR) - 1u) << (lane / LPR * LPR);
  const int wt = p.team, teams = kTeamThreads / 32 / wt, team = warp / wt, tid = threadIdx.x - team * wt * 32;
  const int grp = (warp - team * wt) * RPW + lane / LPR, groups = wt * RPW;
  const int nq = (p.H + groups - 1) / groups, nk = (p.G + groups - 1) / groups, nr = nq + 2 * nk;
  const int half = p.rope >> 1, rest = (HS - p.rope) >> 1, j0 = 4 * l;
  const bool turned = j0 < half;
  const int o1 = turned ? j0 : p.rope + (j0 - half), o2 = o1 + (turned ? half : rest);
  const int hp = min(p.H, kAppParts), gp = min(p.G, kAppParts);
  double* rev = reinterpret_cast<double*>(shared + (size_t)p.stages * nr * COL);
  float2* turns = reinterpret_cast<float2*>(rev + HS / 2) + team * HS;  // [2][HS / 2]
  float* part = reinterpret_cast<float*>(reinterpret_cast<float2*>(rev + HS / 2) + teams * HS) + team * 2 * (hp + gp);
  if ((int)threadIdx.x < half) rev[threadIdx.x] = p.f.rev[threadIdx.x];
  __syncthreads();
  pdl_wait();

  const int64_t step = (int64_t)gridDim.x * teams;
  int64_t tok = (int64_t)blockIdx.x * teams + team;
  constexpr int SIDE = PART == 16 ? kTeamThreads * 16 : 8;
  const int stride = groups * HS;  // from one of the group's rows to the next
  const uint8_t* ring = shared + threadIdx.x * 16;
  const int stage_bytes = nr * COL, koff = nq * COL, voff = (nq + nk) * COL;
  // one group of copies per token, empty behind the last
  const TA *qi = (const TA*)a.q + tok * a.q_stride + grp * HS, *ki = (const TA*)a.k + tok * a.k_stride + grp * HS,
           *vi = (const TA*)a.v + tok * a.v_stride + grp * HS;
  int64_t ti = tok;
  const auto copy = [&](const TA* x, int n, uint32_t dst) {
    for (int h = grp; h < n; h += groups, x += stride, dst += COL) {
      if constexpr (PART == 16) {
        cp_async16_at(dst, x + o1);
        cp_async16_at(dst + SIDE, x + o2);
      } else {
        cp_async8(dst, x + o1);
        cp_async8(dst + SIDE, x + o2);
      }
    }
  };
  const auto issue = [&](const uint8_t* to) {
    if (ti < a.n_tokens) {
      const uint32_t dst = smem_addr(to);
      copy(qi, p.H, dst);
      copy(ki, p.G, dst + koff);
      copy(vi, p.G, dst + voff);
    }
    cp_async_commit();
    ti += step;
    qi += step * a.q_stride;
    ki += step * a.k_stride;
    vi += step * a.v_stride;
  };
  const auto fetch = [&](const uint8_t* src, f2 (&y)[4]) {
    Raw4<TA> r1_, r2_;
    if constexpr (PART == 16) {
      r1_.load(reinterpret_cast<const TA*>(src));
      r2_.load(reinterpret_cast<const TA*>(src + SIDE));
    } else {
      const uint4 w = *reinterpret_cast<const uint4*>(src);
      r1_.w[0] = w.x;
      r1_.w[1] = w.y;
      r2_.w[0] = w.z;
      r2_.w[1] = w.w;
    }
    r1_.get(y);
    r2_.get(y + 2);
  };
  for (int s = 0; s < p.stages; s++) issue(ring + s * stage_bytes);
  const bool fullq = a.q_norm && a.q_norm_len != HS, fullk = a.k_norm && a.k_norm_len != HS;
  int64_t slot = tok < a.n_tokens ? a.slots[tok] : -1;
  int pos = tok < a.n_tokens ? a.pos[tok] : 0;
  TA* qo = (TA*)a.q_out + tok * a.q_out_stride + grp * HS;
  for (int stage = 0, par = 0; tok < a.n_tokens; tok += step, qo += step * a.q_out_stride, par ^= 1) {
    const bool live = slot >= 0 && slot < p.n_slots;
    if (slot >= p.n_slots && tid == 0) set_error(p.err, VIREO_ERR_ARG);
    const int64_t at =
        (live ? (slot >> p.ps_shift) * p.page_stride + (slot & ((1 << p.ps_shift) - 1)) * p.pos_stride : 0) +
        grp * p.head_stride;
    float2* cs = turns + par * (HS / 2);
    float *pq = part + par * (hp + gp), *pk = pq + hp;
    for (int j = tid; j < half; j += 32 * wt) cs[j] = app_angle(pos, rev[j]);
    const int64_t next = tok + step;
    slot = next < a.n_tokens ? a.slots[next] : -1;
    pos = next < a.n_tokens ? a.pos[next] : 0;
    if (p.stages == 2)
      cp_async_wait<1>();
    else
      cp_async_wait<2>();
    const uint8_t* rows = ring + stage * stage_bytes;
    const auto sums = [&](const float* b, int n, const uint8_t* src, float* to) {
      if (b) b += grp * HS;
#pragma unroll 2
      for (int h = grp; h < n; h += groups, src += COL) {
        f2 y[4];
        fetch(src, y);
        if (b) {
          f2 u[4];
          load8(b, o1, o2, u);
          add8(u, y);
          b += stride;
        }
        const float sq = row_sumsq<LPR>(y, mask);
        if (l == 0) put_part(to, h, sq);
      }
    };
    if (fullq) sums(a.bq, p.H, rows, pq);
    if (fullk) sums(a.bk, p.G, rows + koff, pk);
    // angles and sums are written (rows are read and replaced by the same
    // thread, so that in place needs nothing more)
    if (wt == 1)
      __syncwarp();
    else
      asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(32 * wt) : "memory");
    float c[4] = {1.f, 1.f, 1.f, 1.f}, s[4] = {0.f, 0.f, 0.f, 0.f};
    if (turned)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        c[e] = cs[j0 + e].x;
        s[e] = cs[j0 + e].y;
      }
    const auto turn = [&](const float* b, const float* nw, bool full, float f, int n, const uint8_t* src, auto* to,
                          int64_t to_stride) {
      Turn t;
      t.set(c, s, full ? nullptr : nw, o1, o2);
      if (b) b += grp * HS;
      if (full) nw += grp * HS;
#pragma unroll 2
      for (int h = grp; h < n; h += groups, src += COL, to += to_stride) {
        f2 y[4], z[4], u[4];
        if (full) load8(nw, o1, o2, u);
        fetch(src, y);
        if (b) {
          f2 ub[4];
          load8(b, o1, o2, ub);
          add8(ub, y);
          b += stride;
        }
        if (full) {
          mul8(u, y);
          nw += stride;
        } else if (nw) {
          f = rsqrtf(fmaf(row_sumsq<LPR>(y, mask), 1.0f / HS, p.eps));
        }
        t.apply(f, y, z);
        if (!live) continue;
        store4(to + o1, z);
        store4(to + o2, z + 2);
      }
    };
    const float fq = fullq ? rsqrtf(fmaf(sum_parts(pq, p.H), p.per_q, p.eps)) : 1.f;
    const float fk = fullk ? rsqrtf(fmaf(sum_parts(pk, p.G), p.per_k, p.eps)) : 1.f;
    turn(a.bq, a.q_norm, fullq, fq, p.H, rows, qo, stride);
    turn(a.bk, a.k_norm, fullk, fk, p.G, rows + koff, (TC*)p.kc + at, groups * p.head_stride);
    {
      const uint8_t* src = rows + voff;
      TC* vo = (TC*)p.vc + at;
      for (int h = grp; h < p.G; h += groups, src += COL, vo += groups * p.head_stride) {
        f2 y[4];
        fetch(src, y);
        if (a.bv) {
          f2 u[4];
          load8(a.bv + h * HS, o1, o2, u);
          add8(u, y);
        }
        if (!live) continue;
        store4(vo + o1, y);
        store4(vo + o2, y + 2);
      }
    }
    issue(rows);
    stage = stage + 1 < p.stages ? stage + 1 : 0;
  }
}

// Means of the pages whose last position the append wrote: a CTA looks at 32
// tokens' slots for one kv head and sums each page that ends among them with
// all its warps, a lane group per position, in fp32 and in an order that the
// page size alone decides.
constexpr int kMeanTok = 32, kMeanWarps = 8;
template <class TC, int HS>
__global__ void __launch_bounds__(32 * kMeanWarps) kv_means_kernel(const __grid_constant__ AppendParams p) {
  constexpr int E = 16 / (int)sizeof(TC) > HS / 32 ? 16 / (int)sizeof(TC) : HS / 32;
  constexpr int LPR = HS / E, RPW = 32 / LPR;
  __shared__ float sums[kMeanWarps][HS];
  pdl_launch_dependents();
  pdl_wait();
  const int page = 1 << p.ps_shift, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = blockIdx.y;
  const int t = blockIdx.x * kMeanTok + lane;
  const int64_t s = t < p.a.n_tokens ? p.a.slots[t] : -1;
  const bool ends = s >= 0 && s < p.n_slots && (int)(s & (page - 1)) == page - 1;
  const int sub = lane / LPR, l = lane % LPR;
  for (unsigned int m = __ballot_sync(0xffffffffu, ends); m; m &= m - 1) {  // the same in every warp
    const int64_t pg = __shfl_sync(0xffffffffu, s, __ffs(m) - 1) >> p.ps_shift;
    const TC* k = (const TC*)p.kc + pg * p.page_stride + (int64_t)g * p.head_stride + l * E;
    float acc[E];
#pragma unroll
    for (int e = 0; e < E; e++) acc[e] = 0.f;
#pragma unroll 4
    for (int o = warp * RPW + sub; o < page; o += kMeanWarps * RPW) {
      float v[E];
      load_f<E>(k + (int64_t)o * p.pos_stride, v);
#pragma unroll
      for (int e = 0; e < E; e++) acc[e] += v[e];
    }
#pragma unroll
    for (int e = 0; e < E; e++) {
#pragma unroll
      for (int o = LPR; o < 32; o <<= 1) acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], o);
      if (sub == 0) sums[warp][l * E + e] = acc[e];
    }
    __syncthreads();
    for (int d = threadIdx.x; d < HS; d += 32 * kMeanWarps) {
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < kMeanWarps; w++) x += sums[w][d];
      ((TC*)p.a.means)[(pg * p.G + g) * HS + d] = from_f<TC>(x * (1.0f / (float)page));  // exact: a power of two
    }
    __syncthreads();
  }
}

template <class TC, int HS>
static int launch_means(AppendParams& p, cudaStream_t s) {
  if (!p.a.means) return VIREO_OK;
  return pdl_launch(kv_means_kernel<TC, HS>, dim3((p.a.n_tokens + kMeanTok - 1) / kMeanTok, p.G), dim3(32 * kMeanWarps),
                    0, s, p);
}

constexpr size_t kTeamSmem = 104 * 1024;
// Tokens per SM from which on teams take them.  Against a CTA per token, 16 /
// 16 heads of 128 in bf16 and f32 / f16, 400 tokens: 9.2 / 7.1 and 6.9 / 6.9
// us, 2000: 18.8 / 29.0 and 22.1 / 29.4; 32 / 4 of 64, 400: 8.5 / 5.8 and 6.3 /
// 5.8, 2000: 10.1 / 23.3 and 12.5 / 24.2.
constexpr int kTeamTokens = 4;
template <class TA, int HS>
static size_t team_smem(const AppendParams& p) {
  const int groups = p.team * (256 / HS), teams = kTeamThreads / 32 / p.team;
  const size_t nr = (p.H + groups - 1) / groups + 2 * ((p.G + groups - 1) / groups);
  const size_t parts = std::min(p.H, kAppParts) + std::min(p.G, kAppParts);
  return p.stages * nr * 8 * sizeof(TA) * kTeamThreads + (HS / 2) * sizeof(double) +
         teams * (HS * sizeof(float2) + 2 * parts * sizeof(float));
}
// The smallest team with room for two tokens, and for three if there is.  Not
// a whole CTA: with one token at a time it is no better than a CTA per token
// (2000 tokens, 48 / 4 heads of 256, bf16: 56.5 / 45.9 us).
template <class TA, int HS>
static bool team_fits(AppendParams& p) {
  for (p.team = 1; p.team <= kTeamThreads / 64; p.team *= 2)
    for (p.stages = 3; p.stages >= 2; p.stages--)
      if (team_smem<TA, HS>(p) <= kTeamSmem) return true;
  return false;
}

template <class TA, class TC, int HS>
static int launch_append(AppendParams& p, int num_sms, cudaStream_t s) {
  constexpr int GPB = kAppThreads / (HS / 8);
  const gguf_kv_append_args& a = p.a;
  const int rows = p.H + 2 * p.G;
  const bool full = (a.q_norm && a.q_norm_len != HS) || (a.k_norm && a.k_norm_len != HS);
  int64_t blocks;
  if (full) {
    if (a.n_tokens >= kTeamTokens * num_sms && team_fits<TA, HS>(p)) {
      const size_t smem = team_smem<TA, HS>(p);
      int st = cuda_status(cudaFuncSetAttribute(kv_append_team_kernel<TA, TC, HS>,
                                                cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kTeamSmem));
      const int teams = kTeamThreads / 32 / p.team;
      if (!st)
        st = pdl_launch(kv_append_team_kernel<TA, TC, HS>,
                        dim3(std::min(kTeamCtas * num_sms, (a.n_tokens + teams - 1) / teams)), dim3(kTeamThreads), smem,
                        s, p);
      return st ? st : launch_means<TC, HS>(p, s);
    }
    // CTAs to a token: two per SM in all, and one where rows that another CTA
    // sums would be replaced in place
    const int most = (rows + GPB - 1) / GPB;
    p.groups = a.q_out == a.q ? 1 : std::min(most, std::max(1, 2 * num_sms / a.n_tokens));
    p.rpg = (rows + p.groups * GPB - 1) / (p.groups * GPB);
    p.groups = (rows + p.rpg * GPB - 1) / (p.rpg * GPB);
    blocks = (int64_t)a.n_tokens * p.groups;
  } else {
    // as many rows to a lane group as leave about kAppFill CTAs per SM
    const int64_t want = (int64_t)num_sms * kAppFill * GPB;
    p.rpg = (int)std::min<int64_t>(rows, std::max<int64_t>(1, (int64_t)a.n_tokens * rows / want));
    p.groups = (rows + p.rpg - 1) / p.rpg;
    p.rpg = (rows + p.groups - 1) / p.groups;  // evenly
    blocks = ((int64_t)a.n_tokens * p.groups + GPB - 1) / GPB;
  }
  if (blocks > INT32_MAX) return VIREO_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)blocks), block(kAppThreads);
  int st = full                     ? pdl_launch(kv_append_kernel<TA, TC, HS, kAppFull>, grid, block, 0, s, p)
           : a.bq || a.bk || a.bv   ? pdl_launch(kv_append_kernel<TA, TC, HS, kAppBias>, grid, block, 0, s, p)
                                    : pdl_launch(kv_append_kernel<TA, TC, HS, kAppPlain>, grid, block, 0, s, p);
  return st ? st : launch_means<TC, HS>(p, s);
}
template <class TA, class TC>
static int launch_append_h(AppendParams& p, int hs, int num_sms, cudaStream_t s) {
  switch (hs) {
    case 64: return launch_append<TA, TC, 64>(p, num_sms, s);
    case 128: return launch_append<TA, TC, 128>(p, num_sms, s);
    default: return launch_append<TA, TC, 256>(p, num_sms, s);
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
  if (!a || a->n_seqs < 0 || a->n_slots < 0 || a->n_slots > kPlanMaxSlots || a->n_pages < 1 || a->max_pages < 1 ||
      a->page_size < 1 || a->table_stride < a->max_pages || !a->ring || !a->state || !a->cu || !a->state_out ||
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
  // a warp per request (it may end, and give back a row of pages) and a thread
  // per token
  const int items = std::max(a->n_seqs * std::min(32, a->max_pages), a->n_slots);
  const bool in_place = a->kv_len == a->past || a->state_out == a->state;
  const int64_t want = std::max<int64_t>(1, ((int64_t)items + kPlanThreads - 1) / kPlanThreads);
  const bool two = in_place && want > kPlanMaxCluster;
  const int ctas = (int)std::min<int64_t>(4 * c->num_sms, want);
  const int threads = ctas > 1 ? kPlanThreads : std::max(64, (items + 31) / 32 * 32);
  const size_t smem = (size_t)(3 * a->n_seqs + 1) * sizeof(int);
  // 48 KB without asking, less what the kernel has of its own (a few hundred bytes)
  if (smem > 47 * 1024 &&
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
  attr[1].val.clusterDim.x = in_place && !two ? ctas : 1;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  p.part = two ? kPlanTokens : kPlanAll;
  if ((st = cuda_status(cudaLaunchKernelEx(&cfg, kv_plan_kernel, p))) || !two) return st;
  p.part = kPlanLengths;
  cfg.gridDim = dim3(1);
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
  if (a->q_out == a->q && a->q_out_stride != a->q_stride && a->n_tokens > 1) return VIREO_ERR_ARG;
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
  p.per_q = 1.0f / (float)qw;
  p.per_k = 1.0f / (float)kw;
  p.err = c->d_err;
  p.f = kv->freq;
  cudaStream_t s = stream ? (cudaStream_t)stream : c->stream;
  if (d.act_type == KV_BF16) return launch_append_h<__nv_bfloat16, __nv_bfloat16>(p, hs, c->num_sms, s);
  if (d.act_type == KV_F16) return launch_append_h<__half, __half>(p, hs, c->num_sms, s);
  if (d.kv_type == KV_F16) return launch_append_h<float, __half>(p, hs, c->num_sms, s);
  return launch_append_h<float, float>(p, hs, c->num_sms, s);
}

}  // extern "C"
