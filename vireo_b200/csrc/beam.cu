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
// beam_scan_kernel: a CTA goes through a stretch of a row, in chunks that come
// through a ring in shared memory, and leaves a maximum, a sum of exponentials and
// its n_out best tokens.  In the first chunk a bound below the n_out-th best comes
// from the lanes' own maxima: n_out of them are no less than the n_out-th largest
// of a warp's 32, or than what c warps have n_out / c above, and the best of those
// for c = 1, 2, 4, 8 is taken; later it is the n_out-th best so far.  What passes
// is listed, and the list is ranked by counting after chunks 1, 2, 4, 8 ... and
// the last, with no barrier between.  Where it gets more than it holds (equal
// values, rising values), the chunks since the last ranking are read again for
// each of the best.
//
// beam_join_kernel: a CTA per request ranks its lists' best entries, and then the
// entries that are not behind the n_out-th of those.  The sums of exponentials are
// good to kBeamErr of log sum exp in fp32; where two totals of different rows that
// the choice depends on lie nearer than twice that, those rows' sums are taken
// again in 64 bits and the choice is made again.  That costs 51 us for a row of
// 151936 tokens, a 64-bit exponential each in one CTA (eight equal beams 0.43 ms, 32 of
// them 1.6); with totals 0.1 apart it comes once in 100 steps of 32 requests with
// eight beams.  Elsewhere it costs nothing.
//
// 32 requests of 8 beams over 151936 tokens, f32: 45.8 us for both kernels (replayed), 3.4 TB/s,
// floor 24.  Neither HBM (45 %) nor the issue slots (55 %) are at their limit; it is 17
// instructions a logit, where maximum, multiplication, exponential and sum are five.  Rows
// of rising logits list every value: 0.35 ms where random ones take 62 us alone.  Small
// calls are two launches and their latency (one request of 4 beams over 50304: 11.3 us).
// ---------------------------------------------------------------------------
constexpr int kBeamThreads = 256, kBeamWarps = kBeamThreads / 32;
constexpr int kBeamMax = 32;         // beams, and continuations
constexpr int kBeamVocab = 1 << 20;
constexpr int kBeamList = 480;       // candidates, ranked directly with the best so far
constexpr int kBeamJoin = 512;       // threads of the join
constexpr int kBeamLists = 1024;     // stretches of a request's rows, at most
constexpr int kBeamStage = 2048;     // entries of them that the join keeps in shared memory
constexpr int kBeamPerSm = 4;        // CTAs of the pass on an SM
constexpr int kBeamStages = 3;       // of its ring
// Of log sum exp: a chunk's 16 positive terms added in chains of four and a tree
// (6 steps of 2^-24, from there on in 64 bits: 3.6e-7), exp2 (2^-22), and the
// exponent's rounding.  That is half a step of its magnitude; weighed by the
// terms, of which there are at most 2^20, magnitudes are below 20 on average
// (log2(2^20); up to 6 above the reference), and 2^-20 ln(2) is 6.6e-7; the fp32
// log2(e) adds 20 x 1.3e-8.  1.6e-6 in all, below 2^-19.
constexpr double kBeamErr = 0x1p-19;
constexpr float kBeamLog2e = 1.44269504f;
constexpr float kBeamAbove = 4.f;  // of a value above the reference, before a new one is taken

struct BeamParams {
  gguf_beam_args a;
  int splits, chunks;  // stretches of a row, chunks of a stretch
  float* val;    // [rows][splits][n_out] logits of the stretch's best, -inf behind the last
  int* idx;      // their tokens
  double2* stat;  // [rows][splits] reference (-inf: nothing above it), sum of exp(x - reference)
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

// Exponentials are powers of two: e^x as 2^(x l - r), l the fp32 log2(e) and r
// a reference's R l in fp32, in one multiplication and one rounding.  Their sum
// is that of e^x over e^ref, but for (x - R) (l / log2(e) - 1), with this `ref`.
// The largest exponent is what R l lost in its rounding, up to 2^-4 here; of R from
// 2^31 on it could be 128, beyond fp32.  There x - R is formed first, for which the
// values need no more digits than they have, and the reference is R.
VDEV bool beam_far(float R) { return fabsf(R) > 0x1p20f && fabsf(R) < INFINITY; }
VDEV double beam_ref(float R, float r) {
  constexpr double ln2 = 0.69314718055994530942;
  return beam_far(R) ? (double)R : (double)r * ln2 - (double)R * ((double)kBeamLog2e * ln2 - 1.0);
}

VDEV float beam_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// the N-th largest of the warps' values
template <int N>
VDEV float nth(const float* of) {
  float a[N];
#pragma unroll
  for (int i = 0; i < N; i++) a[i] = -INFINITY;
#pragma unroll
  for (int w = 0; w < kBeamWarps; w++) {
    float x = of[w];
#pragma unroll
    for (int i = 0; i < N; i++) {
      const float y = fmaxf(a[i], x);
      x = fminf(a[i], x);
      a[i] = y;
    }
  }
  return a[N - 1];
}

template <class T, int E>
__global__ void __launch_bounds__(kBeamThreads, kBeamPerSm) beam_scan_kernel(const __grid_constant__ BeamParams p) {
  constexpr int VEC = 16 / (int)sizeof(T), NV = E / VEC, CHUNK = kBeamThreads * E;
  __shared__ double red[kBeamWarps], ref[kBeamWarps];
  __shared__ float top[kBeamWarps], thr[4][kBeamWarps];
  __shared__ int counts[2];  // of the list, from one ranking to the next in turn
  __shared__ unsigned long long list[kBeamList + kBeamMax], best[kBeamMax], pick[kBeamWarps];
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
  const int begin = split * p.chunks * CHUNK - lead, end = min(a.vocab, begin + p.chunks * CHUNK);
  // A ring that every thread fills and empties for itself: kBeamPerSm x 48 KB on
  // their way to an SM.  The next chunk in registers was half of that: 83 us where
  // this takes 46.
  extern __shared__ __align__(16) uint4 ring[];  // [kBeamStages][NV][kBeamThreads]
  const auto load = [&](int at, int stage) {  // what lies in the row whole; its ends come with `take`
    if (at < end)
#pragma unroll
      for (int j = 0; j < NV; j++) {
        const int i = at + (j * kBeamThreads + tid) * VEC;
        if (i >= 0 && i + VEC <= a.vocab) cp_async16(&ring[(stage * NV + j) * kBeamThreads + tid], x + i);
      }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  float v[E];
  const auto take = [&](int at, int stage) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kBeamStages - 1) : "memory");
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const int i = at + (j * kBeamThreads + tid) * VEC;
      if (i >= 0 && i + VEC <= a.vocab) {
        const uint4 raw = ring[(stage * NV + j) * kBeamThreads + tid];
        const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int e = 0; e < VEC; e++) v[j * VEC + e] = to_f(t[e]);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; e++) v[j * VEC + e] = i + e >= 0 && i + e < a.vocab ? to_f(x[i + e]) : -INFINITY;
      }
    }
  };
  if (tid < K) best[tid] = 0;
  if (tid == 0) counts[0] = 0;
  int turn = 0, since = begin;  // since: what the list holds begins there
  float R = -INFINITY, from = 0.f;  // this thread's reference, and times log2(e)
  double sum = 0.0;
  float bound = 0.f;  // what a value has to pass, once `full`
  bool full = false;
  int stage = 0;
#pragma unroll
  for (int s = 0; s < kBeamStages; s++) load(begin + s * CHUNK, s);
#pragma unroll 1
  for (int at = begin; at < end; at += CHUNK) {
    take(at, stage);
    load(at + kBeamStages * CHUNK, stage);
    stage = stage == kBeamStages - 1 ? 0 : stage + 1;
    float t4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int e = 0; e < E; e++) t4[e & 3] = fmaxf(t4[e & 3], v[e]);
    const float mine = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3]));
    if (at == begin) {
      // the lanes' maxima in falling order
      float s = mine;
#pragma unroll
      for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int o = size >> 1; o; o >>= 1) {
          const float u = __shfl_xor_sync(0xffffffffu, s, o);
          s = ((lane & size) == 0) == ((lane & o) == 0) ? fmaxf(s, u) : fminf(s, u);
        }
      if (lane == 0) top[warp] = s;
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const float y = __shfl_sync(0xffffffffu, s, (K - 1) >> c);
        if (lane == 0) thr[c][warp] = y;
      }
      __syncthreads();
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < kBeamWarps; w++) M = fmaxf(M, top[w]);
      bound = fmaxf(fmaxf(nth<1>(thr[0]), nth<2>(thr[1])), fmaxf(nth<4>(thr[2]), nth<8>(thr[3])));
      R = M;
      from = M == -INFINITY ? 0.f : M * kBeamLog2e;
    }
    // what passes the bound: at first what reaches it
    const auto passes = [&](float y) { return full ? y > bound : y >= bound && y > -INFINITY; };
    if (passes(mine))
#pragma unroll
      for (int e = 0; e < E; e++)
        if (passes(v[e])) {
          const int n = atomicAdd(&counts[turn], 1), i = at + ((e / VEC) * kBeamThreads + tid) * VEC + e % VEC;
          if (n < kBeamList) list[n] = (unsigned long long)float_key(v[e]) << 32 | (uint32_t)~i;
        }
    // the sum
    if (mine > R + kBeamAbove) {  // also where there is none yet
      if (sum > 0.0) sum *= exp(beam_ref(R, from) - beam_ref(mine, mine * kBeamLog2e));
      R = mine;
      from = mine * kBeamLog2e;
    }
    float s4[4] = {0.f, 0.f, 0.f, 0.f};
    if (beam_far(R)) {
#pragma unroll
      for (int e = 0; e < E; e++) s4[e & 3] += beam_exp2((v[e] - R) * kBeamLog2e);
    } else {
#pragma unroll
      for (int e = 0; e < E; e++) s4[e & 3] += beam_exp2(fmaf(v[e], kBeamLog2e, -from));
    }
    sum += (double)((s4[0] + s4[1]) + (s4[2] + s4[3]));
    const int done = (at - begin) / CHUNK + 1;
    if (at + CHUNK >= end || (done & (done - 1)) == 0) {  // the list with the best so far, ranked
      __syncthreads();
      const int n = counts[turn];
      if (n <= kBeamList) {
        if (tid < K) list[n + tid] = best[tid];
        __syncthreads();
        for (int c = tid; c < n + K; c += kBeamThreads) {
          const unsigned long long key = list[c];
          int rank = 0;
#pragma unroll 4
          for (int o = 0; o < n + K; o++) rank += list[o] > key;
          if (key && rank < K) best[rank] = key;
        }
      } else {  // all of it again, one at a time, each the largest below the last
        unsigned long long last = ~0ull;
        if (tid < K) list[tid] = best[tid];
        int old = 0;  // of the best so far
        for (int k = 0; k < K; k++) {
          unsigned long long key = 0;
          for (int i = max(since, 0) + tid; i < min(a.vocab, at + CHUNK); i += kBeamThreads) {
            const float y = to_f(x[i]);
            const unsigned long long u = y > -INFINITY ? (unsigned long long)float_key(y) << 32 | (uint32_t)~i : 0ull;
            if (u < last && u > key) key = u;
          }
#pragma unroll
          for (int o = 16; o; o >>= 1) {
            const unsigned long long u = __shfl_xor_sync(0xffffffffu, key, o);
            key = u > key ? u : key;
          }
          __syncthreads();
          if (lane == 0) pick[warp] = key;
          __syncthreads();
          for (int w = 0; w < kBeamWarps; w++) key = pick[w] > key ? pick[w] : key;
          if (list[old] > key)
            key = list[old++];
          else
            last = key;
          if (tid == 0) best[k] = key;
        }
      }
      turn ^= 1;
      if (tid == 0) counts[turn] = 0;  // last read before the ranking before this one
      since = at + CHUNK;
      __syncthreads();
      full = best[K - 1] != 0;
      if (full) bound = key_float((uint32_t)(best[K - 1] >> 32));
    }
  }
  // the threads' sums
  const double mine = R == -INFINITY ? -(double)INFINITY : beam_ref(R, from);
  double r = mine;
#pragma unroll
  for (int o = 16; o; o >>= 1) r = fmax(r, __shfl_xor_sync(0xffffffffu, r, o));
  if (lane == 0) ref[warp] = r;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kBeamWarps; w++) r = fmax(r, ref[w]);
  if (r != mine && sum > 0.0) sum *= exp(mine - r);
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) red[warp] = sum;
  __syncthreads();
  const int64_t out = row * p.splits + split;
  if (tid == 0) {
    sum = 0.0;
#pragma unroll
    for (int w = 0; w < kBeamWarps; w++) sum += red[w];
    p.stat[out] = make_double2(r, sum);
  }
  if (tid < K) {
    const unsigned long long key = best[tid];
    p.val[out * K + tid] = key ? key_float((uint32_t)(key >> 32)) : -INFINITY;
    p.idx[out * K + tid] = key ? (int)~(uint32_t)key : -1;
  }
}

struct BeamPick {
  double total;
  int order, list;  // b * vocab + token; the list that it is from
};
// totals in the order of unsigned integers, above 0
VDEV unsigned long long total_key(double v) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(v + 0.0);
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
VDEV double key_total(unsigned long long k) {
  return __longlong_as_double((long long)(k >> 63 ? k & 0x7fffffffffffffffull : ~k));
}

template <class T>
__global__ void __launch_bounds__(kBeamJoin) beam_join_kernel(const __grid_constant__ BeamParams p) {
  constexpr int NW = kBeamJoin / 32;
  __shared__ double lse[kBeamMax], score[kBeamMax], red[NW];
  __shared__ int state[kBeamMax];  // 0: no continuation, 1: over the vocabulary, 2: finished
  __shared__ BeamPick pick[kBeamMax];
  __shared__ unsigned int unsure, near_mask;
  __shared__ uint8_t beam_of[kBeamLists];  // of each list: its row,
  __shared__ int taken[kBeamLists];        // entries taken
  // the lists' best entries, then the candidates
  __shared__ unsigned long long key[kBeamLists], bound;
  __shared__ int order[kBeamLists], bound_order, n_cand;
  __shared__ uint16_t from[kBeamLists], front[kBeamMax];
  static_assert(kBeamMax * kBeamMax <= kBeamLists, "candidates fit");
  __shared__ float sval[kBeamStage];
  __shared__ int sidx[kBeamStage];
  pdl_launch_dependents();
  pdl_wait();
  const gguf_beam_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = a.n_beams, K = a.n_out, S = p.splits;
  const int64_t row0 = (int64_t)blockIdx.x * B;
  const int lists = B * S;
  const bool staged = lists * K <= kBeamStage;
  if (staged)  // rows that were skipped hold anything: nobody looks at them
    for (int e = tid; e < lists * K; e += kBeamJoin) {
      sval[e] = p.val[row0 * S * K + e];
      sidx[e] = p.idx[row0 * S * K + e];
    }
  for (int l = tid; l < lists; l += kBeamJoin) beam_of[l] = (uint8_t)(l / S);
  for (int b = warp; b < B; b += NW) {
    const int64_t row = row0 + b;
    const float sc = a.score[row];
    int st = fabsf(sc) < INFINITY ? (a.done && a.done[row] ? 2 : 1) : 0;
    double l = 0.0;
    if (st == 1) {
      double M = -(double)INFINITY, sum = 0.0;
      for (int s = lane; s < S; s += 32) M = fmax(M, p.stat[row * S + s].x);
#pragma unroll
      for (int o = 16; o; o >>= 1) M = fmax(M, __shfl_xor_sync(0xffffffffu, M, o));
      for (int s = lane; s < S; s += 32) {
        const double2 q = p.stat[row * S + s];
        sum += q.x == M ? q.y : q.y * exp(q.x - M);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      // NaN where a logit is NaN or +inf; 0 where none is above -inf
      if (sum > 0.0 && sum < (double)INFINITY && M < (double)INFINITY)
        l = M + log(sum);
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
  // the h-th of a list, 0 where there is none
  const auto entry = [&](int l, int h, int& o) {
    const int b = beam_of[l];
    o = INT32_MAX;
    if (state[b] == 1 && h < K) {
      const int e = l * K + h;
      const float x = staged ? sval[e] : p.val[row0 * S * K + e];
      if (x > -INFINITY) {
        o = b * a.vocab + (staged ? sidx[e] : p.idx[row0 * S * K + e]);
        return total_key(score[b] + (double)x - lse[b]);
      }
    } else if (state[b] == 2 && h == 0 && l == b * S) {
      o = b * a.vocab + a.end_token;
      return total_key(score[b]);
    }
    return 0ull;
  };
  int found = 0;
  for (int pass = 0;; pass++) {
    // The K best lists by their best entries; only what is not behind the last of
    // those can be among the K best of all, and that is at most K entries of each.
    if (tid == 0) {
      unsure = near_mask = 0;
      bound = 0;
      n_cand = 0;
    }
    if (tid < K) front[tid] = 0xffff;
    for (int l = tid; l < lists; l += kBeamJoin) taken[l] = 0;
    // h entries of each of K / h lists are K as well: with many asked for, a higher bound
    for (int h = 1; h == 1 || (h <= 4 && K >= 16); h *= 2) {
      for (int l = tid; l < lists; l += kBeamJoin) key[l] = entry(l, h - 1, order[l]);
      __syncthreads();
      for (int l = tid; l < lists; l += kBeamJoin) {
        // equal ones in the lists' order: those of one row rise in tokens, rows in b
        const unsigned long long k = key[l];
        const int l0 = l & ~31, l1 = min(l0 + 32, lists);
        int rank = 0;
#pragma unroll 8
        for (int x = 0; x < l0; x++) rank += key[x] >= k;
#pragma unroll 8
        for (int x = l0; x < l1; x++) rank += key[x] > k || (key[x] == k && x < l);
#pragma unroll 8
        for (int x = l1; x < lists; x++) rank += key[x] > k;
        if (k && h == 1 && rank < K) front[rank] = (uint16_t)l;
        // of equal totals the lists' order tells at h = 1 alone: further down an entry before
        // the h-th, of a higher logit, may round to the same total and have the larger token
        if (rank == (K - 1) / h && k > bound) {
          bound = k;
          bound_order = h == 1 ? order[l] : INT32_MAX;
        }
      }
      __syncthreads();
    }
    for (int x = tid; x < K * K; x += kBeamJoin) {
      const int l = front[x / K];
      if (l == 0xffff) break;
      int o;
      const unsigned long long k = entry(l, x % K, o);
      if (k && (k > bound || (k == bound && o <= bound_order))) {
        const int n = atomicAdd(&n_cand, 1);
        key[n] = k;
        order[n] = o;
        from[n] = (uint16_t)l;
      }
    }
    __syncthreads();
    const int n = n_cand;
    found = min(n, K);
    for (int c = tid; c < n; c += kBeamJoin) {
      const unsigned long long k = key[c];
      const int o = order[c];
      int rank = 0;
#pragma unroll 4
      for (int x = 0; x < n; x++) rank += key[x] > k || (key[x] == k && order[x] < o);
      if (rank < K) {
        pick[rank] = {key_total(k), o, from[c]};
        atomicAdd(&taken[from[c]], 1);
      }
    }
    __syncthreads();
    if (pass) break;
    // What lies too near a total of another row: neighbours among the picks,
    // and heads that are left near the last pick.
    if (found == K) {
      const double last = pick[K - 1].total;
      for (int l = tid; l < lists; l += kBeamJoin) {
        int o;
        const unsigned long long k = entry(l, taken[l], o);
        if (k && key_total(k) >= last - 2 * kBeamErr) atomicOr(&near_mask, 1u << beam_of[l]);
      }
    }
    __syncthreads();
    if (tid == 0) {
      unsigned int mask = 0, rest = near_mask;
      for (int k = 0; k + 1 < found; k++) {
        const int x = beam_of[pick[k].list], y = beam_of[pick[k + 1].list];
        if (x != y && pick[k].total - pick[k + 1].total <= 2 * kBeamErr) mask |= 1u << x | 1u << y;
      }
      if (rest) {
        for (int k = 0; k < found; k++)
          if (pick[k].total <= pick[found - 1].total + 2 * kBeamErr) rest |= 1u << beam_of[pick[k].list];
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
      double M = -(double)INFINITY;
      for (int s = 0; s < S; s++) M = fmax(M, p.stat[(row0 + b) * S + s].x);
      double sum = 0.0;
#pragma unroll 1
      for (int i0 = tid; i0 < a.vocab; i0 += 16 * kBeamJoin) {
        float y[16];  // on their way together
#pragma unroll
        for (int e = 0; e < 16; e++) y[e] = i0 + e * kBeamJoin < a.vocab ? to_f(x[i0 + e * kBeamJoin]) : -INFINITY;
#pragma unroll 4
        for (int e = 0; e < 16; e++) sum += exp((double)y[e] - M);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) red[warp] = sum;
      __syncthreads();
      if (tid == 0) {
        for (int w = 1; w < NW; w++) sum += red[w];
        lse[b] = M + log(sum);
      }
      __syncthreads();
    }
  }
  __syncthreads();
  if (tid < K) {
    const int64_t o = (int64_t)blockIdx.x * K + tid;
    const bool there = tid < found;
    const int b = there ? beam_of[pick[tid].list] : 0, token = there ? pick[tid].order - b * a.vocab : -1;
    a.score_out[o] = there ? (float)pick[tid].total : -INFINITY;
    a.token[o] = token;
    a.parent[o] = there ? (int)(row0 + b) : -1;
    if (a.done_out) a.done_out[o] = !there || token == a.end_token;
  }
}

// How a row is cut: values of a thread in a chunk, stretches, chunks of one.
// Small calls take a chunk of half the size to a CTA, to have more of them;
// others about as many CTAs as the GPU holds, or a multiple of that: of 1 to 16
// stretches the fewest whose last wave is at least 85 % full, else the best.
struct BeamCut {
  int each, splits, chunks;
};
static BeamCut beam_cut(int64_t rows, int beams, int vocab, int num_sms) {
  const auto chunks_of = [&](int each) { return (vocab + 7 + kBeamThreads * each - 1) / (kBeamThreads * each); };
  const int64_t held = (int64_t)num_sms * kBeamPerSm;
  const int most = kBeamLists / beams;
  BeamCut c = {16, 1, chunks_of(16)};
  if (rows * chunks_of(16) <= held) {
    if (rows * chunks_of(8) <= held && chunks_of(8) <= most) c.each = 8;
    c.splits = std::min(most, chunks_of(c.each));
  } else {
    double best = 0.0;
    for (int s = 1; s <= std::min({16, most, chunks_of(16)}) && best < 0.85; s++) {
      const int per = (chunks_of(16) + s - 1) / s, used = (chunks_of(16) + per - 1) / per;
      const int64_t ctas = rows * used, waves = (ctas + held - 1) / held;
      // of the whole: full waves, and stretches of one length
      const double full = (double)ctas / (double)(waves * held) * chunks_of(16) / ((double)used * per);
      if (full > best) {
        best = full;
        c.splits = used;
      }
    }
    // few rows: whatever spreads them over the GPU
    if (rows * c.splits < held / 2) c.splits = std::min<int64_t>({most, chunks_of(16), (held + rows - 1) / rows});
  }
  c.chunks = (chunks_of(c.each) + c.splits - 1) / c.splits;
  c.splits = (chunks_of(c.each) + c.chunks - 1) / c.chunks;
  return c;
}

static size_t beam_up(size_t v) { return (v + 255) & ~(size_t)255; }

template <class T>
static int beam_launch(const BeamParams& p, int each, cudaStream_t s) {
  const dim3 grid((unsigned)((int64_t)p.a.n_seqs * p.a.n_beams * p.splits)), block(kBeamThreads);
  const size_t smem = (size_t)kBeamStages * kBeamThreads * each * sizeof(T);
  int st = each == 16 ? cuda_status(cudaFuncSetAttribute(beam_scan_kernel<T, 16>,
                                                         cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem))
                      : VIREO_OK;
  if (st) return st;
  st = each == 16 ? pdl_launch(beam_scan_kernel<T, 16>, grid, block, smem, s, p)
                  : pdl_launch(beam_scan_kernel<T, 8>, grid, block, smem, s, p);
  return st ? st : pdl_launch(beam_join_kernel<T>, dim3(p.a.n_seqs), dim3(kBeamJoin), 0, s, p);
}

}  // namespace vireo

using namespace vireo;

extern "C" {

size_t gguf_beam_workspace(int n_seqs, int n_beams, int n_out, int vocab) {
  if (n_seqs < 0 || n_beams < 1 || n_beams > kBeamMax || n_out < 1 || n_out > kBeamMax || vocab < 1 ||
      vocab > kBeamVocab)
    return 0;
  // the most stretches that a call may choose
  const int64_t stretches =
      (int64_t)n_seqs * n_beams * std::min(kBeamLists / n_beams, (vocab + 7 + kBeamThreads * 8 - 1) / (kBeamThreads * 8));
  return 2 * beam_up((size_t)stretches * n_out * 4) + beam_up((size_t)stretches * sizeof(double2));
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
  if (rows * kBeamLists > INT32_MAX) return VIREO_ERR_UNSUPPORTED;
  int st;
  Ctx* c = ctx_get(&st);
  if (!c) return st;
  DeviceGuard dg(c->device);
  if (dg.status) return dg.status;
  BeamParams p;
  p.a = *a;
  const BeamCut cut = beam_cut(rows, a->n_beams, a->vocab, c->num_sms);
  const int each = cut.each;
  p.splits = cut.splits;
  p.chunks = cut.chunks;
  const size_t lists = beam_up((size_t)rows * cut.splits * a->n_out * 4);
  p.val = (float*)a->ws;
  p.idx = (int*)((uint8_t*)a->ws + lists);
  p.stat = (double2*)((uint8_t*)a->ws + 2 * lists);
  cudaStream_t s = stream ? (cudaStream_t)stream : c->stream;
  if (a->type == KV_BF16) return beam_launch<__nv_bfloat16>(p, each, s);
  if (a->type == KV_F16) return beam_launch<__half>(p, each, s);
  return beam_launch<float>(p, each, s);
}

}  // extern "C"
