// The choice of a beam search's continuations (include/gguf_beam.h): one pass
// over the logits, then a join per request.
#include <math.h>

#include "gguf_beam.h"
#include "paged_kv.cuh"
#include "pdl_launch.cuh"

namespace vireo {

// ---------------------------------------------------------------------------
// Within a row the totals are ordered as the logits are, so a row's best
// n_out tokens need no logarithm; between rows it is log sum exp that decides.
//
// beam_scan_kernel: a CTA takes a stretch of a row into registers, and leaves
// its maximum, its sum of exponentials and its n_out best tokens.  A bound
// below the n_out-th best comes from the lanes' own maxima: the n_out-th
// largest of a warp's 32, the best of the warps'.  What reaches it (a few
// dozen) is listed and ranked by counting; where more than the list holds do
// (a row of equal values), they are taken one at a time.
//
// beam_join_kernel: a CTA per request takes the best heads of its lists in
// turn.  The sums of exponentials are good to kBeamErr of log sum exp in
// fp32; where two totals of different rows that the choice depends on lie
// nearer than twice that, those rows' sums are taken again in 64 bits and the
// choice is made again.  That costs about 50 us a row where it happens (in a
// step of 32 requests with eight beams about once in 100) and nothing
// elsewhere, where 64 bits throughout would double the time of the pass.
//
// The pass is bound by HBM: 4 bytes and about eight instructions a logit.
// ---------------------------------------------------------------------------
constexpr int kBeamThreads = 256, kBeamWarps = kBeamThreads / 32;
constexpr int kBeamMax = 32;         // beams, and continuations
constexpr int kBeamVocab = 1 << 20;
constexpr int kBeamList = 512;       // candidates of a stretch, ranked directly
constexpr int kBeamJoin = 512;       // threads of the join
constexpr int kBeamLists = 4128;     // stretches of a request's rows: 32 rows of 2^20 / 8192 + 1
// Of log sum exp: adding up to 32 + 8 + 128 positive terms in trees and short
// chains (18 steps of 2^-24 to the end, then 64 bits), exp2 (2^-22), and the
// rounding of x - max, which weighs (max - x) 2^-25 and by entropy at most
// ln(2^20) 2^-25 over the sum: 1.8e-6 in all, below 2^-19.
constexpr double kBeamErr = 0x1p-19;

struct BeamParams {
  gguf_beam_args a;
  int splits;
  float* val;    // [rows][splits][n_out] logits of the stretch's best, -inf behind the last
  int* idx;      // their tokens
  float2* stat;  // [rows][splits] maximum, sum of exp(x - maximum)
};

// floats in the order of unsigned integers, -0 as 0
VDEV uint32_t float_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  return v != v ? 0u : u & 0x80000000u ? ~u : u | 0x80000000u;
}
VDEV float key_float(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

VDEV bool beam_live(const gguf_beam_args& a, int64_t row) {
  const float s = a.score[row];
  return fabsf(s) < INFINITY && !(a.done && a.done[row]);
}

// e^d for d <= 0 (0 for -inf): exp2 of d log2(e), with what the product's
// rounding lost
VDEV float exp_below(float d) {
  const float t = d * 1.44269504f;
  const float c = fmaf(d, 1.44269504f, -t) + d * 1.925963e-8f;
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(t));
  return t > -126.f ? fmaf(y, c * 0.69314718f, y) : y;
}

template <class T, int E>
__global__ void __launch_bounds__(kBeamThreads) beam_scan_kernel(const __grid_constant__ BeamParams p) {
  constexpr int VEC = 16 / (int)sizeof(T), CHUNK = kBeamThreads * E;
  __shared__ float red[kBeamWarps], thr[kBeamWarps];
  __shared__ int count;
  __shared__ unsigned long long list[kBeamList];
  pdl_launch_dependents();
  pdl_wait();
  const gguf_beam_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = a.n_out;
  const int64_t row = blockIdx.x / p.splits;
  const int split = (int)(blockIdx.x - row * p.splits);
  if (!beam_live(a, row)) return;
  const T* x = reinterpret_cast<const T*>(a.logits) + row * a.stride;
  // places are counted from the 16-byte boundary at or before the row
  const int lead = (int)(((uintptr_t)x & 15) / sizeof(T));
  const int at = split * CHUNK + tid * VEC - lead;
  float v[E];
#pragma unroll
  for (int j = 0; j < E / VEC; j++) {
    const int i = at + j * kBeamThreads * VEC;
    if (i >= 0 && i + VEC <= a.vocab) {
      float t[VEC];
      load_f<VEC>(x + i, t);
#pragma unroll
      for (int e = 0; e < VEC; e++) v[j * VEC + e] = t[e];
    } else {
#pragma unroll
      for (int e = 0; e < VEC; e++) v[j * VEC + e] = i + e >= 0 && i + e < a.vocab ? to_f(x[i + e]) : -INFINITY;
    }
  }
  if (tid == 0) count = 0;
  float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int e = 0; e < E; e++) top[e & 3] = fmaxf(top[e & 3], v[e]);
  const float mine = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
  // the lanes' maxima in falling order
  float s = mine;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int o = size >> 1; o; o >>= 1) {
      const float u = __shfl_xor_sync(0xffffffffu, s, o);
      s = ((lane & size) == 0) == ((lane & o) == 0) ? fmaxf(s, u) : fminf(s, u);
    }
  const float wmax = __shfl_sync(0xffffffffu, s, 0), wth = __shfl_sync(0xffffffffu, s, K - 1);
  if (lane == 0) {
    red[warp] = wmax;
    thr[warp] = wth;
  }
  __syncthreads();
  float M = -INFINITY, T0 = -INFINITY;
#pragma unroll
  for (int w = 0; w < kBeamWarps; w++) {
    M = fmaxf(M, red[w]);
    T0 = fmaxf(T0, thr[w]);
  }
  // what reaches the bound
#pragma unroll
  for (int e = 0; e < E; e++)
    if (v[e] >= T0 && v[e] > -INFINITY) {
      const int n = atomicAdd(&count, 1);
      const int i = at + (e / VEC) * kBeamThreads * VEC + e % VEC;
      if (n < kBeamList) list[n] = (unsigned long long)float_key(v[e]) << 32 | (uint32_t)~i;
    }
  // the sum
  const float m = M == -INFINITY ? 0.f : M;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < E; e++) sum[e & 3] += exp_below(v[e] - m);
  float total = (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
  for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  __syncthreads();  // the list is complete, and the maxima are read
  if (lane == 0) red[warp] = total;
  const int n = count;
  const int64_t out = (row * p.splits + split) * K;
  if (n <= kBeamList) {
    for (int c = tid; c < n; c += kBeamThreads) {
      const unsigned long long key = list[c];
      int rank = 0;
      for (int o = 0; o < n; o++) rank += list[o] > key;
      if (rank < K) {
        p.val[out + rank] = key_float((uint32_t)(key >> 32));
        p.idx[out + rank] = (int)~(uint32_t)key;
      }
    }
    if (tid < K && tid >= n) {
      p.val[out + tid] = -INFINITY;
      p.idx[out + tid] = -1;
    }
  } else {  // one at a time, each the largest below the last
    unsigned long long last = ~0ull;
    for (int k = 0; k < K; k++) {
      unsigned long long best = 0;
#pragma unroll
      for (int e = 0; e < E; e++) {
        const int i = at + (e / VEC) * kBeamThreads * VEC + e % VEC;
        const unsigned long long key =
            v[e] > -INFINITY ? (unsigned long long)float_key(v[e]) << 32 | (uint32_t)~i : 0ull;
        if (key < last && key > best) best = key;
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        const unsigned long long u = __shfl_xor_sync(0xffffffffu, best, o);
        best = u > best ? u : best;
      }
      __syncthreads();
      if (lane == 0) list[warp] = best;
      __syncthreads();
      for (int w = 0; w < kBeamWarps; w++) best = list[w] > best ? list[w] : best;
      last = best;
      if (tid == 0) {
        p.val[out + k] = best ? key_float((uint32_t)(best >> 32)) : -INFINITY;
        p.idx[out + k] = best ? (int)~(uint32_t)best : -1;
      }
    }
  }
  __syncthreads();
  if (tid == 0) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kBeamWarps; w++) t += red[w];
    p.stat[row * p.splits + split] = make_float2(M, t);
  }
}

struct BeamPick {
  double total;
  int order, list;  // b * vocab + token; the list it heads, or -1 of nothing
};
VDEV bool before(const BeamPick& x, const BeamPick& y) {
  return x.total > y.total || (x.total == y.total && x.order < y.order);
}

template <class T>
__global__ void __launch_bounds__(kBeamJoin) beam_join_kernel(const __grid_constant__ BeamParams p) {
  constexpr int NW = kBeamJoin / 32;
  __shared__ double lse[kBeamMax], score[kBeamMax], red[NW];
  __shared__ int state[kBeamMax];  // 0: no continuation, 1: over the vocabulary, 2: finished
  __shared__ BeamPick best[2][NW], pick[kBeamMax];
  __shared__ unsigned int unsure, near_mask;
  __shared__ uint8_t head[kBeamLists];
  pdl_launch_dependents();
  pdl_wait();
  const gguf_beam_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = a.n_beams, K = a.n_out, S = p.splits;
  const int64_t row0 = (int64_t)blockIdx.x * B;
  for (int b = warp; b < B; b += NW) {
    const int64_t row = row0 + b;
    const float sc = a.score[row];
    int st = fabsf(sc) < INFINITY ? (a.done && a.done[row] ? 2 : 1) : 0;
    double l = 0.0;
    if (st == 1) {
      float M = -INFINITY;
      for (int s = lane; s < S; s += 32) M = fmaxf(M, p.stat[row * S + s].x);
#pragma unroll
      for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
      double sum = 0.0;
      for (int s = lane; s < S; s += 32) {
        const float2 q = p.stat[row * S + s];
        if (q.x > -INFINITY || q.y != 0.f) sum += (double)q.y * exp((double)q.x - (double)M);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      // NaN where a logit is NaN or +inf; no maximum where none is finite
      if (fabsf(M) < INFINITY && sum > 0.0 && sum < (double)INFINITY)
        l = (double)M + log(sum);
      else
        st = 0;
    }
    if (lane == 0) {
      state[b] = st;
      lse[b] = l;
      score[b] = (double)sc;
    }
  }
  __syncthreads();
  const int lists = B * S;
  const auto entry = [&](int l, int h) {
    BeamPick q = {-(double)INFINITY, INT32_MAX, -1};
    const int b = l / S;
    if (state[b] == 1 && h < K) {
      const int64_t e = (row0 * S + l) * K + h;
      const float x = p.val[e];
      if (x > -INFINITY) q = {score[b] + (double)x - lse[b], b * a.vocab + p.idx[e], l};
    } else if (state[b] == 2 && h == 0 && l == b * S) {
      q = {score[b], b * a.vocab + a.end_token, l};
    }
    return q;
  };
  int found = 0;
  for (int pass = 0;; pass++) {
    for (int l = tid; l < lists; l += kBeamJoin) head[l] = 0;
    if (tid == 0) unsure = near_mask = 0;
    // the best of this thread's lists
    BeamPick mine = {-(double)INFINITY, INT32_MAX, -1};
    const auto look = [&]() {
      mine = {-(double)INFINITY, INT32_MAX, -1};
      for (int l = tid; l < lists; l += kBeamJoin) {
        const BeamPick q = entry(l, head[l]);
        if (before(q, mine)) mine = q;
      }
    };
    look();
    for (found = 0; found < K; found++) {
      BeamPick q = mine;
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        BeamPick u;
        u.total = __shfl_xor_sync(0xffffffffu, q.total, o);
        u.order = __shfl_xor_sync(0xffffffffu, q.order, o);
        u.list = __shfl_xor_sync(0xffffffffu, q.list, o);
        if (before(u, q)) q = u;
      }
      if (lane == 0) best[found & 1][warp] = q;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NW; w++)
        if (before(best[found & 1][w], q)) q = best[found & 1][w];
      if (q.list < 0) break;
      if (tid == 0) pick[found] = q;
      if (q.list % kBeamJoin == tid) {
        head[q.list]++;
        look();
      }
    }
    if (pass) break;
    __syncthreads();
    // What lies too near a total of another row: neighbours among the picks,
    // and heads that are left near the last pick.
    if (found == K) {
      const double last = pick[K - 1].total;
      for (int l = tid; l < lists; l += kBeamJoin) {
        const BeamPick q = entry(l, head[l]);
        if (q.list >= 0 && q.total >= last - 2 * kBeamErr) atomicOr(&near_mask, 1u << (l / S));
      }
    }
    __syncthreads();
    if (tid == 0) {
      unsigned int mask = 0, rest = near_mask;
      for (int k = 0; k + 1 < found; k++) {
        const int x = pick[k].list / S, y = pick[k + 1].list / S;
        if (x != y && pick[k].total - pick[k + 1].total <= 2 * kBeamErr) mask |= 1u << x | 1u << y;
      }
      if (rest) {
        for (int k = 0; k < found; k++)
          if (pick[k].total <= pick[found - 1].total + 2 * kBeamErr) rest |= 1u << (pick[k].list / S);
        if (rest & (rest - 1)) mask |= rest;
      }
      // a finished row's total is exact
      for (int b = 0; b < B; b++)
        if (state[b] != 1) mask &= ~(1u << b);
      unsure = mask;
    }
    __syncthreads();
    unsigned int mask = unsure;
    if (!mask) break;
    for (; mask; mask &= mask - 1) {
      const int b = __ffs(mask) - 1;
      const T* x = reinterpret_cast<const T*>(a.logits) + (row0 + b) * a.stride;
      float M = -INFINITY;
      for (int s = 0; s < S; s++) M = fmaxf(M, p.stat[(row0 + b) * S + s].x);
      double sum = 0.0;
#pragma unroll 4
      for (int i = tid; i < a.vocab; i += kBeamJoin) sum += exp((double)to_f(x[i]) - (double)M);
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) red[warp] = sum;
      __syncthreads();
      if (tid == 0) {
        for (int w = 1; w < NW; w++) sum += red[w];
        lse[b] = (double)M + log(sum);
      }
      __syncthreads();
    }
  }
  __syncthreads();
  if (tid < K) {
    const int64_t o = (int64_t)blockIdx.x * K + tid;
    const bool there = tid < found;
    const int b = there ? pick[tid].list / S : 0, token = there ? pick[tid].order - b * a.vocab : -1;
    a.score_out[o] = there ? (float)pick[tid].total : -INFINITY;
    a.token[o] = token;
    a.parent[o] = there ? (int)(row0 + b) : -1;
    if (a.done_out) a.done_out[o] = !there || token == a.end_token;
  }
}

// Values of a thread: 32, or fewer where that leaves SMs idle.
static int beam_each(int64_t rows, int beams, int vocab, int num_sms) {
  int e = 32;
  while (e > 8 && rows * ((vocab + kBeamThreads * e - 1) / (kBeamThreads * e)) < 2 * num_sms &&
         (int64_t)beams * ((vocab + 7 + kBeamThreads * e / 2 - 1) / (kBeamThreads * e / 2)) <= kBeamLists)
    e /= 2;
  return e;
}
static int beam_splits(int vocab, int each) { return (vocab + 7 + kBeamThreads * each - 1) / (kBeamThreads * each); }

static size_t beam_up(size_t v) { return (v + 255) & ~(size_t)255; }

template <class T>
static int beam_launch(const BeamParams& p, int each, cudaStream_t s) {
  const dim3 grid((unsigned)((int64_t)p.a.n_seqs * p.a.n_beams * p.splits)), block(kBeamThreads);
  const int st = each == 32   ? pdl_launch(beam_scan_kernel<T, 32>, grid, block, 0, s, p)
                 : each == 16 ? pdl_launch(beam_scan_kernel<T, 16>, grid, block, 0, s, p)
                              : pdl_launch(beam_scan_kernel<T, 8>, grid, block, 0, s, p);
  return st ? st : pdl_launch(beam_join_kernel<T>, dim3(p.a.n_seqs), dim3(kBeamJoin), 0, s, p);
}

}  // namespace vireo

using namespace vireo;

extern "C" {

size_t gguf_beam_workspace(int n_seqs, int n_beams, int n_out, int vocab) {
  if (n_seqs < 0 || n_beams < 1 || n_beams > kBeamMax || n_out < 1 || n_out > kBeamMax || vocab < 1 ||
      vocab > kBeamVocab)
    return 0;
  // the smallest stretches that a call may choose
  const int64_t stretches = (int64_t)n_seqs * n_beams * beam_splits(vocab, 8);
  return 2 * beam_up((size_t)stretches * n_out * 4) + beam_up((size_t)stretches * sizeof(float2));
}

int gguf_beam_select(const gguf_beam_args* a, void* stream) {
  if (!a || a->n_seqs < 0 || a->n_beams < 1 || a->n_out < 1 || a->vocab < 1 ||
      (int64_t)a->n_beams * a->vocab < a->n_out || a->end_token < -1 || a->end_token >= a->vocab ||
      (a->done && a->end_token < 0))
    return VIREO_ERR_ARG;
  if (a->n_beams > kBeamMax || a->n_out > kBeamMax || a->vocab > kBeamVocab ||
      (a->type != KV_F32 && a->type != KV_F16 && a->type != KV_BF16))
    return VIREO_ERR_UNSUPPORTED;
  if (a->n_seqs == 0) return VIREO_OK;
  const int64_t rows = (int64_t)a->n_seqs * a->n_beams;
  if (!a->logits || !kv_aligned(a->logits, kv_type_size(a->type)) || !a->score || !a->score_out || !a->token ||
      !a->parent || !a->ws || !kv_aligned(a->ws, 256) ||
      (rows > 1 && (a->stride < a->vocab || a->stride > (INT64_MAX >> 6) / rows)) ||
      a->ws_bytes < gguf_beam_workspace(a->n_seqs, a->n_beams, a->n_out, a->vocab))
    return VIREO_ERR_ARG;
  if (rows * beam_splits(a->vocab, 8) > INT32_MAX) return VIREO_ERR_UNSUPPORTED;
  int st;
  Ctx* c = ctx_get(&st);
  if (!c) return st;
  DeviceGuard dg(c->device);
  if (dg.status) return dg.status;
  BeamParams p;
  p.a = *a;
  const int each = beam_each(rows, a->n_beams, a->vocab, c->num_sms);
  p.splits = beam_splits(a->vocab, each);
  const size_t lists = beam_up((size_t)rows * beam_splits(a->vocab, 8) * a->n_out * 4);
  p.val = (float*)a->ws;
  p.idx = (int*)((uint8_t*)a->ws + lists);
  p.stat = (float2*)((uint8_t*)a->ws + 2 * lists);
  cudaStream_t s = stream ? (cudaStream_t)stream : c->stream;
  if (a->type == KV_BF16) return beam_launch<__nv_bfloat16>(p, each, s);
  if (a->type == KV_F16) return beam_launch<__half>(p, each, s);
  return beam_launch<float>(p, each, s);
}

}  // extern "C"
