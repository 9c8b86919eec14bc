// Attention of one new token per request over the paged key-value pool
// (include/gguf_kv.h): over every cached position, or over pages that a
// cheap score selects.
//
// out = softmax(scale q . K) V per (request, q head).  The cache is read
// once, so the call is bound by HBM: 2 * head_size values per position and
// kv head against about four operations per value and q head.  Three things
// follow.
//
//  * Work is cut evenly, whatever the lengths.  The positions of all
//    (request, kv head) pairs, in tiles, form one line; CTA i of a grid that
//    fills the GPU once takes the i-th equal stretch of it.  A pair that lies
//    inside one CTA is finished there; a pair that several CTAs share leaves
//    one partial state (accumulator, running maximum, running sum) per CTA,
//    at most two partial states per CTA in all, so the workspace is as large
//    as the GPU and not as the batch.  kv_merge_kernel joins them.
//  * The copies never wait for the arithmetic: two producer warps, one for
//    keys and one for values, walk the tiles with TMA (a 4-D tensor map per
//    pool: dimension, position, head, page; one box per page and 128 bytes of
//    a row, 128-byte swizzle) into a ring of stages.  A warp starts a box in
//    about 140 cycles, its lanes one after the other: boxes of 1 KB (pages of
//    8 positions) from one warp per CTA reach 4.2 TB/s, from two 5.7.  A page
//    number outside the pool is out of the map's bounds and reads as zeros.
//  * The arithmetic is small enough for mma.sync: up to eight q heads of a kv
//    head are the rows 0-7 of the M side.  Rows 8-15 would be empty; they hold
//    what rounding to the cache's type lost (of q where it is fp32, of the
//    softmax weights always), so both products keep about twice the type's
//    digits (22 with f16, 16 with bf16) at no further instruction, and the
//    two halves are added in fp32.  With an f16 cache weights are held 2^14
//    times as large, which keeps those digits down to weights of 2^-17 and
//    leaves an absolute error of 2^-39 below; a key that outweighs thousands
//    of others would otherwise drop them from the output, not from the sum.
//    An fp32 cache runs on the CUDA cores in plain fp32.
//
// Softmax weights are powers of two of scores scaled by log2(e), with the
// running maximum and sum in fp32.
//
// Measured (per call, replayed): 64 ragged requests of up to 8192 positions,
// 4 kv heads of 128, bf16, 550 MB: 92 us, 0.92 of the copy bandwidth.  The same
// geometry in f32 / f16, one request: both launches with nothing to do 2.5
// us; one tile in one CTA, nothing to join 5.2; one tile in each of 148 CTAs,
// joined 7.5; each further tile 0.5 to 0.9 (four 9.7); stretches that end
// inside other pairs, two states to a CTA, 1 more (8200 positions, 3.5 tiles to
// a CTA: 10.5).
#include <limits.h>
#include <math.h>

#include <cmath>
#include <type_traits>

#include "paged_kv.cuh"
#include "pdl_launch.cuh"

namespace vireo {

constexpr int kPaHeads = 8;  // q heads of a warp's products
// Consumer warps, and two producers: one for keys, one for values.  A warp
// takes 16 positions of a tile (8 of an fp32 one), so a stage is 32 KB for 64
// and for 128 dimensions; twice the warps at 64 dimensions because a warp's
// share of a tile costs it nearly the same number of instructions at half the
// bytes.
template <int HS>
__host__ __device__ constexpr int kv_warps() { return HS == 64 ? 8 : 4; }
// SG: groups of consumer warps, each with eight heads of the unit's and all of
// its tiles.  More than eight heads to a kv head take two groups, so that
// the cache is read once for all sixteen (at 256 dimensions their
// accumulators leave no registers for it, and the cache is read again).
template <int HS, int SG>
__host__ __device__ constexpr int kv_threads() { return 32 * (kv_warps<HS>() * SG + 2); }
constexpr int kPaMaxWarps = 18;
template <int HS>
__host__ __device__ constexpr int kv_state_row() { return HS == 64 ? HS + 2 : HS + 4; }
constexpr float kLog2e = 1.4426950408889634f;

template <class TC, int HS>
__host__ __device__ constexpr int kv_tile() { return kv_warps<HS>() * (sizeof(TC) == 4 ? 8 : 16); }
template <class TC, int HS>
__host__ __device__ constexpr int kv_stage_bytes() { return 2 * kv_tile<TC, HS>() * HS * (int)sizeof(TC); }
// stages of the ring: 96 KB in flight per CTA (192 KB at 256 dimensions), two
// CTAs to an SM up to 128 dimensions, so that the copies of one run under the
// joins of the other
constexpr int kPaStages = 3;
// tiles whose products are added up on the tensor cores
constexpr int kPaRun = 32;

struct KvAttnParams {
  const void* q;
  void* out;
  int64_t q_stride, out_stride, table_stride;
  const int32_t* table;  // block tables, or with nsel the chosen pages [n_seqs][G][nsel], physical
  const int32_t* kv_len;
  int n_seqs, max_pages, n_pages;
  int H, G, R, nsub;     // q heads, kv heads, heads per kv head, units per kv head
  int heads;             // q heads a unit takes, at most: 8 or 16
  int ps_shift, nsel, ctas, sms;
  int whole;             // a CTA per pair, nothing to join
  int small;             // the line's length fits 31 bits
  float scale;           // times log2(e)
  float* part;           // [ctas][2][heads][HS + 4]: accumulator, maximum, sum
  int2* where;           // [n_seqs][G][nsub] of pairs with positions: 2 x first CTA + its state, CTAs; null with `whole`
  int* err;
};

// cached positions of a request as the kernels see them, and, with block
// selection, the positions on its chosen pages
VDEV int kv_len_of(const KvAttnParams& p, int seq) {
  int n = max(p.kv_len[seq], 0);
  const int most = p.max_pages << p.ps_shift;
  if (n > most) {
    set_error(p.err, VIREO_ERR_ARG);
    n = most;
  }
  if (p.nsel) {
    const int np = (n + (1 << p.ps_shift) - 1) >> p.ps_shift;
    if (np > p.nsel) n -= (np - p.nsel) << p.ps_shift;
  }
  return n;
}

// The line of tiles cut over the CTAs: a request's units start at (tiles of
// the requests before it) x (kv heads x subs), each (kv head, sub) in turn.
// CTAs that get a stretch: all that fit on the GPU where each then has a
// ring's worth of tiles, else one per SM; the partial states to join would
// cost more than the second CTA of an SM saves.  One request of 8200
// positions, 516 tiles: 10.2 us with 148 CTAs, 11.8 with 296.
VDEV int cut_ctas(const KvAttnParams& p, long long total) {
  return total >= (long long)kPaStages * p.ctas ? p.ctas : (int)min((long long)min(p.sms, p.ctas), total);
}
VDEV int div_cut(int a, int b) { return (int)((uint32_t)a / (uint32_t)b); }  // both >= 0
VDEV long long div_cut(long long a, long long b) { return a / b; }
// CTA i takes units [at(i), at(i + 1)): q each, the first r of them one more
template <class I>
struct KvCut {
  I q;
  int r;
  VDEV KvCut(I total, int ctas) {
    q = div_cut(total, (I)ctas);
    r = (int)(total - q * ctas);
  }
  VDEV I at(int i) const { return q * i + min(i, r); }
};

// a producer's or consumer's place on the line
template <int TILE>
struct KvWalk {
  int seq, kh, sub, tile, len, ntile;
  long long left;  // tiles left in this CTA's stretch
  VDEV void load(const KvAttnParams& p) {
    len = kv_len_of(p, seq);
    ntile = (len + TILE - 1) / TILE;
  }
  // tiles of the current pair that belong to this CTA
  VDEV int count() const { return (int)min((long long)(ntile - tile), left); }
  VDEV void next(const KvAttnParams& p) {  // past the current pair's tiles
    left -= count();
    tile = 0;
    if (left <= 0 || ++sub < p.nsub) return;
    sub = 0;
    if (++kh < p.G) return;
    kh = 0;
    do {
      seq++;
      load(p);
    } while (ntile == 0 && seq + 1 < p.n_seqs);  // left > 0: a request with tiles follows
    if (ntile == 0) left = 0;
  }
};

// The shared state that kernel and producer agree on.
struct KvRing {
  uint64_t full[kPaStages], empty[kPaStages];
  long long red[kPaMaxWarps];
  long long cut_q;  // the cut, as in KvCut
  int cut_r;
  int found[5];
  int abort;
};

// Finds the CTA's stretch: block-wide, every thread returns the same walk.
// I: the type of places on the line (64-bit scans and divisions cost a CTA
// about 0.4 us of its start).
template <class I, int TILE, int NWARP>
VDEV KvWalk<TILE> kv_start(const KvAttnParams& p, KvRing* ring) {
  I* red = reinterpret_cast<I*>(ring->red);
  constexpr int nt = 32 * NWARP;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int units = p.G * p.nsub;
  const int per = p.n_seqs <= nt ? 1 : (p.n_seqs + nt - 1) / nt;
  const int lo = min(p.n_seqs, tid * per), hi = min(p.n_seqs, lo + per);
  const int len0 = lo < hi ? kv_len_of(p, lo) : 0;
  I sum = (len0 + TILE - 1) / TILE;
  for (int s = lo + 1; s < hi; s++) sum += (kv_len_of(p, s) + TILE - 1) / TILE;
  I inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const I u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 31) red[warp] = inc;
  __syncthreads();
  I before = inc - sum, total = 0;
#pragma unroll
  for (int w = 0; w < NWARP; w++) {
    const I v = red[w];
    if (w < warp) before += v;
    total += v;
  }
  total *= units;
  KvWalk<TILE> k;
  const int ctas = total ? cut_ctas(p, total) : 0;
  k.left = 0;
  k.seq = k.kh = k.sub = k.tile = k.len = k.ntile = 0;
  if ((int)blockIdx.x >= ctas) return k;
  const KvCut<I> cut(total, ctas);
  const I u0 = cut.at(blockIdx.x);
  if (u0 >= before * units && u0 < (before + sum) * units) {  // one thread
    I b = before * units;
    for (int s = lo; s < hi; s++) {
      const int len = s == lo ? len0 : kv_len_of(p, s), n = (len + TILE - 1) / TILE;
      if (u0 < b + (I)n * units) {
        const int unit = (int)div_cut(u0 - b, (I)n), kh = unit / p.nsub;
        ring->found[0] = s;
        ring->found[1] = kh;
        ring->found[2] = unit - kh * p.nsub;
        ring->found[3] = (int)(u0 - b - (I)unit * n);
        ring->found[4] = len;
        ring->cut_q = cut.q;
        ring->cut_r = cut.r;
        break;
      }
      b += (I)n * units;
    }
  }
  __syncthreads();
  k.seq = ring->found[0];
  k.kh = ring->found[1];
  k.sub = ring->found[2];
  k.tile = ring->found[3];
  k.len = ring->found[4];
  k.ntile = (k.len + TILE - 1) / TILE;
  k.left = cut.at(blockIdx.x + 1) - u0;
  return k;
}

// 2^x to 2^-22 of itself; weights below 2^-126 are zero
VDEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A pair to a CTA.
template <int TILE>
VDEV KvWalk<TILE> kv_pair(const KvAttnParams& p) {
  KvWalk<TILE> k;
  const int units = p.G * p.nsub, unit = blockIdx.x % units;
  k.seq = blockIdx.x / units;
  k.kh = unit / p.nsub;
  k.sub = unit - k.kh * p.nsub;
  k.tile = 0;
  k.load(p);
  k.left = k.ntile;
  return k;
}

VDEV void ldsm4(uint32_t row, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(row)
               : "memory");
}
VDEV void ldsm4_trans(uint32_t row, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(row)
               : "memory");
}
VDEV void mma_kv(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) { mma_16816(d, a, b0, b1); }
VDEV void mma_kv(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// two values rounded to the cache's type, and what the rounding lost
VDEV uint32_t pack2(float a, float b, __half) { return pack_h2(a, b); }
VDEV uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
VDEV float2 unpack2(uint32_t u, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
VDEV float2 unpack2(uint32_t u, __nv_bfloat16) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u));
}
template <class TC>
VDEV uint32_t pack2_rest(uint32_t hi, float a, float b) {
  const float2 f = unpack2(hi, TC());
  return pack2(a - f.x, b - f.y, TC());
}

// Every lane waits for itself: one try when the phase is done.
VDEV bool mbar_wait_lanes(uint64_t* bar, uint32_t parity, const volatile int* abort) {
  const bool ok = mbar_test(bar, parity) || mbar_wait(bar, parity, abort);
  return __all_sync(0xffffffffu, ok);
}
// a place in the ring: stage and phase
struct KvSlot {
  int i = 0;
  uint32_t phase = 0;
  VDEV void next() {
    if (++i == kPaStages) {
      i = 0;
      phase ^= 1u;
    }
  }
};

// A weight 2^x of the products, x <= 0.  f16 holds nothing finer than 2^-24,
// so there weights reach up to 2^14 instead of 1; sums carry the same factor
// and the division by them takes it out.  (Added to the difference: added to
// the maximum it could be lost or doubled in the rounding of a large one.)
template <class TC>
VDEV float weight(float x) {
  if constexpr (std::is_same_v<TC, __half>) x += 14.f;
  return ex2(x);
}

// a product and that of the rests; an infinite one stands for itself (its
// rest is an infinity of either sign, or NaN)
VDEV float add_rest(float v, float rest) { return fabsf(v) < INFINITY ? v + rest : v; }

// the next pair's q rows into L1 while this pair runs
template <class TA, int HS, int TILE>
VDEV void prefetch_q(const KvAttnParams& p, const KvWalk<TILE>& w) {
  KvWalk<TILE> nx = w;
  nx.next(p);
  if (nx.left <= 0) return;
  const int nh = min(p.heads, p.R - nx.sub * p.heads);
  const TA* q = reinterpret_cast<const TA*>(p.q) + (int64_t)nx.seq * p.q_stride +
                (int64_t)(nx.kh * p.R + nx.sub * p.heads) * HS;
  const int at = (int)threadIdx.x * 128;
  uint32_t line;
  if (at < nh * HS * (int)sizeof(TA))
    asm volatile("ld.global.ca.b32 %0, [%1];" : "=r"(line) : "l"(reinterpret_cast<const uint8_t*>(q) + at));
}

// the warps of one group
template <int HS>
VDEV void consumer_sync(int sg) { asm volatile("bar.sync %0, %1;" ::"r"(1 + sg), "r"(32 * kv_warps<HS>()) : "memory"); }

// CTAs that share a pair of n tiles whose first `here` are the last of this
// CTA's stretch
VDEV int kv_sharers(const KvRing* ring, int n, int here) {
  long long rest = n - here;
  const long long q = ring->cut_q;
  const int b = (int)blockIdx.x + 1, wide = max(0, ring->cut_r - b);  // CTAs after this one with q + 1
  if (rest <= 0) return 1;
  if (rest <= (q + 1) * wide) return 1 + (int)((rest + q) / (q + 1));
  rest -= (q + 1) * wide;
  return 1 + wide + (int)((rest + q - 1) / q);
}

// ---- producer warps ----------------------------------------------------------
// one pool's half of every stage; `where`, if given, is told where the states
// of the pairs are that start in this CTA
template <class TC, int HS>
VDEV void kv_produce(const KvAttnParams& p, const CUtensorMap* map, KvWalk<kv_tile<TC, HS>()> w, KvRing* ring,
                     uint8_t* stages, int2* where) {
  constexpr int TILE = kv_tile<TC, HS>(), NB = HS * (int)sizeof(TC) / 128, XE = 128 / (int)sizeof(TC);
  constexpr int BOX = TILE * 128;  // bytes of one 128-byte column of a tile
  const int lane = threadIdx.x & 31;
  const int page = 1 << p.ps_shift, ppt = max(1, TILE >> p.ps_shift), rows = min(page, TILE);
  int it = 0;
  KvSlot sl;
  // Page numbers are read 32 at a time, a window ahead of the one in use, and
  // the next pair's first window with this pair's: a number read when its
  // tile is due would put its latency between any two tiles.
  const auto pages_of = [&](const KvWalk<TILE>& x, int first) {  // pages first .. first + 31 of x's pair
    const int i = first + lane;
    const int32_t* row =
        p.nsel ? p.table + ((int64_t)x.seq * p.G + x.kh) * p.nsel : p.table + (int64_t)x.seq * p.table_stride;
    return i < (x.len + page - 1) >> p.ps_shift ? row[i] : 0;
  };
  int win = pages_of(w, w.tile * TILE >> p.ps_shift);
  int state = 2 * blockIdx.x;  // the CTA's first pair leaves its first state, a later one its second
  for (; w.left > 0; state = 2 * blockIdx.x + 1) {
    KvWalk<TILE> nx = w;
    nx.next(p);
    const int g = w.kh, n = w.count(), npages = (w.len + page - 1) >> p.ps_shift;
    int base = w.tile * TILE >> p.ps_shift;
    int ahead = pages_of(w, base + 32);
    const int nwin = nx.left > 0 ? pages_of(nx, nx.tile * TILE >> p.ps_shift) : 0;
    for (int t = w.tile; t < w.tile + n; t++, it++, sl.next()) {
      const int p0 = t * TILE >> p.ps_shift;
      if (p0 - base >= 32) {
        base += 32;
        win = ahead;
        ahead = pages_of(w, base + 32);
      }
      const int mpi = p0 + (lane & (ppt - 1));
      const int mine = __shfl_sync(0xffffffffu, win, mpi - base);
      const bool has = lane < ppt && mpi < npages;
      const int cnt = __popc(__ballot_sync(0xffffffffu, has));
      const int slot = sl.i;
      if (it >= kPaStages && !mbar_wait_lanes(&ring->empty[slot], sl.phase ^ 1u, &ring->abort)) goto drain;
      if (lane == 0) mbar_arrive_expect_tx(&ring->full[slot], (uint32_t)(cnt * rows * HS * (int)sizeof(TC)));
      __syncwarp();
      if (has) {
        int pg = mine;
        if (pg < 0 || pg >= p.n_pages) {
          set_error(p.err, VIREO_ERR_ARG);
          pg = p.n_pages;  // outside the map: zeros
        }
        const int off = (t * TILE) & (page - 1);  // 0 when a tile holds whole pages
        uint8_t* dst = stages + (size_t)slot * kv_stage_bytes<TC, HS>() + lane * rows * 128;
#pragma unroll
        for (int b = 0; b < NB; b++) tma_load_4d(dst + b * BOX, map, b * XE, off, g, pg, &ring->full[slot]);
      }
    }
    if (where && lane == 0 && w.tile == 0)
      where[((int64_t)w.seq * p.G + g) * p.nsub + w.sub] = make_int2(state, kv_sharers(ring, w.ntile, n));
    w = nx;
    win = nwin;
  }
drain:
  // no copy may still be landing when the CTA exits
  {
    const int never = 0;
    for (int j = it > kPaStages ? it - kPaStages : 0; j < it; j++)
      mbar_wait_warp(&ring->full[j % kPaStages], (uint32_t)(j / kPaStages) & 1u, &never);
  }
}

// where a (row, 16-byte chunk) of a swizzled tile lies: rows of 128 bytes in
// columns of TILE rows, the chunk XORed with the row
template <int TILE>
VDEV uint32_t kv_at(int r, int c) {
  return (uint32_t)((c >> 3) * TILE * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// shared floats: the warps' states, and what the fp32 path for up to four
// heads keeps beside them
template <class TC, int HS, int RT, int SG>
__host__ __device__ constexpr int kv_merge_floats() {
  constexpr int states = (kv_warps<HS>() * RT * kv_state_row<HS>() + 3) / 4 * 4;
  return SG * (states + (sizeof(TC) == 4 && RT < kPaHeads ? RT * HS + kv_warps<HS>() * 8 * RT : 0));
}
template <class TC, int HS, int RT, int SG>
constexpr int kv_attn_smem() {
  return kPaStages * kv_stage_bytes<TC, HS>() + kv_merge_floats<TC, HS, RT, SG>() * 4 + (int)sizeof(KvRing);
}

// ---- the warps' states joined --------------------------------------------------
// Every warp has put its state of each head, [NW][RT][HS + 4] (HS + 2 at 64
// dimensions, where eight warps' states must leave room for a second CTA on
// the SM): accumulator, maximum, sum.  All threads of the group then take a
// share of one head's dimensions, finish the pair if this CTA had all of its
// tiles, else leave one partial state.
template <class TA, int HS, int RT>
VDEV void kv_join(const KvAttnParams& p, const float* merge, int tid, int seq, int h0, int sg, int nh, bool whole,
                  int slot) {
  constexpr int NW = kv_warps<HS>(), V = HS == 64 ? 2 : 4, ROW = kv_state_row<HS>();
  constexpr int TPH = 32 * NW / RT < HS / V ? 32 * NW / RT : HS / V;  // threads per head, V dimensions at a time
  constexpr int NV = HS / (V * TPH);
  const int h = tid / TPH, t = tid % TPH;
  if (h >= nh) return;
  const float* st = merge + h * ROW;
  float m[NW], M = -INFINITY, L = 0.f;
#pragma unroll
  for (int w = 0; w < NW; w++) {
    m[w] = st[w * RT * ROW + HS];
    M = fmaxf(M, m[w]);
  }
  const float m_sub = M == -INFINITY ? 0.f : M;  // scores of -inf alone
#pragma unroll
  for (int w = 0; w < NW; w++) {
    m[w] = ex2(m[w] - m_sub);
    L += m[w] * st[w * RT * ROW + HS + 1];
  }
  float o[NV][V];
#pragma unroll
  for (int c = 0; c < NV; c++)
#pragma unroll
    for (int e = 0; e < V; e++) o[c][e] = 0.f;
#pragma unroll
  for (int w = 0; w < NW; w++)
#pragma unroll
    for (int c = 0; c < NV; c++) {
      float v[V];
      load_f<V>(st + w * RT * ROW + V * (t + TPH * c), v);
#pragma unroll
      for (int e = 0; e < V; e++) o[c][e] += v[e] * m[w];
    }
  if (whole) {
    const float r = L > 0.f ? 1.0f / L : (L == 0.f ? 0.f : L);  // a NaN stays one
    TA* out = reinterpret_cast<TA*>(p.out) + (int64_t)seq * p.out_stride + (int64_t)(h0 + h) * HS;
#pragma unroll
    for (int c = 0; c < NV; c++) {
#pragma unroll
      for (int e = 0; e < V; e++) o[c][e] *= r;
      store_f<V>(out + V * (t + TPH * c), o[c]);
    }
  } else {
    float* b = p.part + ((size_t)(2 * blockIdx.x + slot) * p.heads + sg * kPaHeads + h) * (HS + 4);
#pragma unroll
    for (int c = 0; c < NV; c++) store_f<V>(b + V * (t + TPH * c), o[c]);
    if (t == 0) {
      b[HS] = M;
      b[HS + 1] = L;
    }
  }
}

// ---- 16-bit cache: tensor cores ------------------------------------------------
// The products' accumulators round towards zero, and a sum of one sign loses
// 2^-24 of itself a step or so: 1e-4 over 65,536 positions of a pair in one CTA.
// So the tiles are taken in runs of kPaRun, and what a run leaves is added to
// the warp's state in shared memory, rounded to nearest (2e-6 at any length).
// RUNS: whether a CTA can get more than one run of a pair; the code for it
// costs the others 0.3 to 0.5 us a call (one request of 8200 positions, 32 / 4
// heads of 128: 11.0 us with it, 10.5 without).
template <class TA, class TC, int HS, int SG, bool RUNS>
VDEV void kv_consume_mma(const KvAttnParams& p, KvWalk<kv_tile<TC, HS>()> w, KvRing* ring, uint8_t* stages,
                         float* merge) {
  constexpr int TILE = kv_tile<TC, HS>(), KS = HS / 16, NT = HS / 8, NW = kv_warps<HS>();
  constexpr bool QSPLIT = sizeof(TA) == 4;
  const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int sg = SG == 1 ? 0 : (int)(threadIdx.x >> 5) / NW;  // the group, and the warp in it
  const int warp = (int)(threadIdx.x >> 5) - sg * NW;
  merge += sg * NW * kPaHeads * kv_state_row<HS>();
  const int wr = 16 * warp;  // this warp's rows of a tile
  // A lane's ldmatrix rows in a stage.  Its row's position in the swizzle is
  // r7 throughout, so chunk c of the row is where chunk 0 is with the low
  // three bits of c XORed in, in column c / 8: two addresses for the keys (a
  // step of four chunks), four for the values (steps of two), and constants.
  const uint32_t r7 = lane & 7, base = smem_addr(stages);
  const uint32_t k_at = base + (wr + r7) * 128 + (((lane >> 3) ^ r7) << 4);
  const uint32_t v_at =
      base + TILE * HS * 2 + (wr + r7 + 8 * ((lane >> 3) & 1)) * 128 + (((lane >> 4) ^ r7) << 4);
  KvSlot sl;
  for (bool first = true; w.left > 0; w.next(p), first = false) {
    const int kh = w.kh, sub = w.sub, n = w.count();
    const int first_h = sub * p.heads + sg * kPaHeads, nh = min(kPaHeads, p.R - first_h);  // 0 or less: none
    const int h = kh * p.R + first_h + g;  // this lane's q head, if g < nh
    // q as A fragments: row g the value in the cache's type, row g + 8 what
    // that left of an fp32 value.  An fp32 row is first scaled by the power
    // of two that brings its largest value to [2^14, 2^15), as far up as f16
    // goes: values down to 2^-17 of the largest keep 22 bits, smaller ones
    // are off by 2^-39 of it at most.  The scores take the power back.
    uint32_t qa[KS][QSPLIT ? 4 : 2];
    float qs = p.scale;
    {
      const TA* q = reinterpret_cast<const TA*>(p.q) + (int64_t)w.seq * p.q_stride + (int64_t)h * HS;
      if constexpr (QSPLIT) {
        float v[KS][4];
        float mx = 0.f;
#pragma unroll
        for (int s = 0; s < KS; s++) {
          float2 a = make_float2(0.f, 0.f), b = a;
          if (g < nh) {
            a = *reinterpret_cast<const float2*>(q + 16 * s + 2 * t4);
            b = *reinterpret_cast<const float2*>(q + 16 * s + 8 + 2 * t4);
          }
          v[s][0] = a.x;
          v[s][1] = a.y;
          v[s][2] = b.x;
          v[s][3] = b.y;
          mx = fmaxf(fmaxf(fmaxf(mx, fabsf(a.x)), fmaxf(fabsf(a.y), fabsf(b.x))), fabsf(b.y));
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // within what a power of two and its inverse can hold; beside an
        // infinity no finite value may become one
        const int e = mx > 0.f ? min(max(ilogbf(mx), -112), 127) - 14 : 0;
        const float down = ldexpf(1.f, -e);
        qs *= ldexpf(1.f, e);
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
          for (int j = 0; j < 2; j++) {
            const float a = v[s][2 * j] * down, b = v[s][2 * j + 1] * down;
            qa[s][2 * j] = pack2(a, b, TC());
            qa[s][2 * j + 1] = pack2_rest<TC>(qa[s][2 * j], a, b);
          }
      } else {
#pragma unroll
        for (int s = 0; s < KS; s++) {
          qa[s][0] = g < nh ? *reinterpret_cast<const uint32_t*>(q + 16 * s + 2 * t4) : 0u;
          qa[s][1] = g < nh ? *reinterpret_cast<const uint32_t*>(q + 16 * s + 8 + 2 * t4) : 0u;
        }
      }
    }
    prefetch_q<TA, HS>(p, w);
    float* st = merge + (warp * kPaHeads + g) * kv_state_row<HS>();
    float o[NT][4];
#pragma unroll
    for (int j = 0; j < NT; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    float m_run = -INFINITY, l_run = 0.f;
    const int end = w.tile + n;
    int stop = RUNS ? min(end, w.tile + kPaRun) : end;
#pragma unroll 1
    for (int t = w.tile;;) {
      if (t == stop) {
        l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
        l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);
#pragma unroll
        for (int j = 0; j < NT; j++) {
          o[j][0] = add_rest(o[j][0], o[j][2]);
          o[j][1] = add_rest(o[j][1], o[j][3]);
        }
        if (!RUNS || t - w.tile <= kPaRun) {
          consumer_sync<HS>(sg);  // the last pair's states are read
        } else {
          const float f = ex2(st[HS] - (m_run == -INFINITY ? 0.f : m_run));
          l_run = fmaf(st[HS + 1], f, l_run);
#pragma unroll
          for (int j = 0; j < NT; j++) {
            const float2 x = *reinterpret_cast<const float2*>(st + 8 * j + 2 * t4);
            o[j][0] = fmaf(x.x, f, o[j][0]);
            o[j][1] = fmaf(x.y, f, o[j][1]);
          }
          __syncwarp();
        }
#pragma unroll
        for (int j = 0; j < NT; j++) *reinterpret_cast<float2*>(st + 8 * j + 2 * t4) = make_float2(o[j][0], o[j][1]);
        if (t4 == 0) {
          st[HS] = m_run;
          st[HS + 1] = l_run;
        }
        if (!RUNS || t == end) break;
        __syncwarp();
        l_run = 0.f;
        stop = min(end, t + kPaRun);
#pragma unroll
        for (int j = 0; j < NT; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
      }
      const bool ok = mbar_wait_lanes(&ring->full[sl.i], sl.phase, &ring->abort);
      if (!ok && lane == 0) {
        ring->abort = 1;
        set_error(p.err, VIREO_ERR_TIMEOUT);
      }
      const uint32_t stage = (uint32_t)sl.i * kv_stage_bytes<TC, HS>();
      const int rows = w.len - t * TILE;  // of this tile, or more
      if (ok && wr < rows && nh > 0) {
        const bool part = wr + 16 > rows;
        if (part) {
          // value rows behind the last position: zeros, since their weight of
          // zero does not cancel a NaN
          uint8_t* vt = stages + stage + TILE * HS * 2;
          for (int r = rows; r < wr + 16; r++)
            for (int c = lane; c < HS / 8; c += 32)
              *reinterpret_cast<uint4*>(vt + kv_at<TILE>(r, c)) = make_uint4(0u, 0u, 0u, 0u);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the stage is filled by copies again
          __syncwarp();
        }
        const uint32_t ka[2] = {k_at + stage, (k_at ^ 64u) + stage};
        // two sums each, of the even and of the odd steps: half the chain of
        // dependent products
        float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f}, u0[4] = {0.f, 0.f, 0.f, 0.f},
              u1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < KS; s += 2) {
          uint32_t b[2][4];
#pragma unroll
          for (int j = 0; j < 2; j++)
            ldsm4(ka[(s >> 1) & 1] + (s >> 2) * TILE * 128 + j * 1024, b[j][0], b[j][1], b[j][2], b[j][3]);
          uint32_t a0[4], a1[4];
          if constexpr (QSPLIT) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
              a0[i] = qa[s][i];
              a1[i] = qa[s + 1][i];
            }
          } else {
            a0[0] = qa[s][0];
            a0[2] = qa[s][1];
            a1[0] = qa[s + 1][0];
            a1[2] = qa[s + 1][1];
            a0[1] = a0[3] = a1[1] = a1[3] = 0u;
          }
          mma_kv(s0, a0, b[0][0], b[0][1], TC());
          mma_kv(s1, a0, b[1][0], b[1][1], TC());
          mma_kv(u0, a1, b[0][2], b[0][3], TC());
          mma_kv(u1, a1, b[1][2], b[1][3], TC());
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
          s0[i] += u0[i];
          s1[i] += u1[i];
        }
        if constexpr (QSPLIT) {
          s0[0] = add_rest(s0[0], s0[2]);
          s0[1] = add_rest(s0[1], s0[3]);
          s1[0] = add_rest(s1[0], s1[2]);
          s1[1] = add_rest(s1[1], s1[3]);
        }
        // this lane's positions: wr + 2 t4 (+1) and wr + 8 + 2 t4 (+1)
        float v0 = s0[0] * qs, v1 = s0[1] * qs, v2 = s1[0] * qs, v3 = s1[1] * qs;
        if (part) {
          const int q0 = wr + 2 * t4;
          v0 = q0 < rows ? v0 : -INFINITY;
          v1 = q0 + 1 < rows ? v1 : -INFINITY;
          v2 = q0 + 8 < rows ? v2 : -INFINITY;
          v3 = q0 + 9 < rows ? v3 : -INFINITY;
        }
        float mt = fmaxf(fmaxf(v0, v1), fmaxf(v2, v3));
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
        const float m_new = fmaxf(m_run, mt);
        // scores of -inf alone leave the maximum at -inf: subtract 0 then
        const float m_sub = m_new == -INFINITY ? 0.f : m_new;
        if (__any_sync(0xffffffffu, m_new > m_run)) {
          const float alpha = ex2(m_run - m_sub);
          l_run *= alpha;
#pragma unroll
          for (int j = 0; j < NT; j++) {
            o[j][0] *= alpha;
            o[j][1] *= alpha;
            o[j][2] *= alpha;
            o[j][3] *= alpha;
          }
          m_run = m_new;
        }
        const float e0 = weight<TC>(v0 - m_sub), e1 = weight<TC>(v1 - m_sub), e2 = weight<TC>(v2 - m_sub),
                    e3 = weight<TC>(v3 - m_sub);
        l_run += (e0 + e1) + (e2 + e3);
        uint32_t pa[4];
        pa[0] = pack2(e0, e1, TC());
        pa[1] = pack2_rest<TC>(pa[0], e0, e1);
        pa[2] = pack2(e2, e3, TC());
        pa[3] = pack2_rest<TC>(pa[2], e2, e3);
#pragma unroll
        for (int j = 0; j < NT; j += 2) {
          uint32_t b0, b1, b2, b3;
          ldsm4_trans((v_at ^ ((j & 7) << 4)) + stage + (j >> 3) * TILE * 128, b0, b1, b2, b3);
          mma_kv(o[j], pa, b0, b1, TC());
          mma_kv(o[j + 1], pa, b2, b3, TC());
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&ring->empty[sl.i]);
      sl.next();
      t++;
    }
    consumer_sync<HS>(sg);
    kv_join<TA, HS, kPaHeads>(p, merge, threadIdx.x - 32 * NW * sg, w.seq, kh * p.R + first_h, sg, nh,
                              w.tile == 0 && n == w.ntile, first ? 0 : 1);
  }
}

// ---- fp32 cache: CUDA cores ----------------------------------------------------
// A warp takes eight of a tile's positions.
//
// Up to four heads.  Scores: lane (position lane & 7, quarter lane >> 3)
// multiplies every fourth 16-byte chunk of its key with the RT q heads in
// shared memory; the quarters are added by shuffles.  Values: lane i owns
// 16-byte chunk i (mod chunks of a row) of the output and adds weight x value
// over the positions.
template <int HS, int RT>
VDEV void kv_consume_f32(const KvAttnParams& p, KvWalk<kv_tile<float, HS>()> w, KvRing* ring, uint8_t* stages,
                         float* merge) {
  constexpr int TILE = kv_tile<float, HS>(), CH = HS / 4, NW = kv_warps<HS>();  // CH: chunks of a row
  constexpr int PS = CH < 32 ? 32 / CH : 1, NC = CH < 32 ? 1 : CH / 32;  // positions side by side, chunks per lane
  const int lane = threadIdx.x & 31, pp = lane & 7, qd = lane >> 3;
  const int tid = threadIdx.x, warp = tid >> 5;
  float* sq = merge + (NW * RT * kv_state_row<HS>() + 3) / 4 * 4;  // [RT][HS], behind the warps' states
  float* sp = sq + RT * HS + warp * 8 * RT;                        // the warp's weights, [8][RT]
  KvSlot sl;
  const int wr = 8 * warp;
  const uint32_t k_at = (wr + pp) * 128 + ((qd ^ pp) << 4);  // chunks 4 i + qd of row wr + pp: as for the tensor cores
  for (bool first = true; w.left > 0; w.next(p), first = false) {
    const int kh = w.kh, sub = w.sub, n = w.count();
    const int first_h = sub * p.heads, nh = min(RT, p.R - first_h), h0 = kh * p.R + first_h;
    const float* q = reinterpret_cast<const float*>(p.q) + (int64_t)w.seq * p.q_stride + (int64_t)h0 * HS;
    for (int i = tid * 4; i < RT * HS; i += 32 * NW * 4)
      *reinterpret_cast<float4*>(sq + i) =
          i < nh * HS ? *reinterpret_cast<const float4*>(q + i) : make_float4(0.f, 0.f, 0.f, 0.f);
    consumer_sync<HS>(0);
    prefetch_q<float, HS>(p, w);
    float o[RT][NC * 4], m_run[RT], l_run[RT];
#pragma unroll
    for (int r = 0; r < RT; r++) {
      m_run[r] = -INFINITY;
      l_run[r] = 0.f;
#pragma unroll
      for (int j = 0; j < NC * 4; j++) o[r][j] = 0.f;
    }
#pragma unroll 1
    for (int t = w.tile; t < w.tile + n; t++, sl.next()) {
      const bool ok = mbar_wait_lanes(&ring->full[sl.i], sl.phase, &ring->abort);
      if (!ok && lane == 0) {
        ring->abort = 1;
        set_error(p.err, VIREO_ERR_TIMEOUT);
      }
      const uint8_t* kt = stages + (size_t)sl.i * kv_stage_bytes<float, HS>();
      const uint8_t* vt = kt + TILE * HS * 4;
      const int rows = min(TILE, w.len - t * TILE);
      if (ok && wr < rows && nh > 0) {
        float s[RT];
#pragma unroll
        for (int r = 0; r < RT; r++) s[r] = 0.f;
#pragma unroll
        for (int i = 0; i < CH / 4; i++) {
          const int c = 4 * i + qd;
          const float4 k = *reinterpret_cast<const float4*>(kt + (k_at ^ (i & 1) * 64) + (i >> 1) * TILE * 128);
#pragma unroll
          for (int r = 0; r < RT; r++) {
            const float4 x = *reinterpret_cast<const float4*>(sq + r * HS + 4 * c);
            s[r] += x.x * k.x;
            s[r] += x.y * k.y;
            s[r] += x.z * k.z;
            s[r] += x.w * k.w;
          }
        }
        const bool live = wr + pp < rows;
        bool up = false;
        float m_old[RT];
#pragma unroll
        for (int r = 0; r < RT; r++) {
          s[r] += __shfl_xor_sync(0xffffffffu, s[r], 8);
          s[r] += __shfl_xor_sync(0xffffffffu, s[r], 16);
          s[r] = live ? s[r] * p.scale : -INFINITY;
          float m = s[r];
#pragma unroll
          for (int x = 1; x < 8; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
          m_old[r] = m_run[r];
          up |= m > m_run[r];
          m_run[r] = fmaxf(m_run[r], m);
        }
        if (up) {  // the same in every lane
#pragma unroll
          for (int r = 0; r < RT; r++) {
            const float a = ex2(m_old[r] - (m_run[r] == -INFINITY ? 0.f : m_run[r]));
            l_run[r] *= a;
#pragma unroll
            for (int j = 0; j < NC * 4; j++) o[r][j] *= a;
          }
        }
#pragma unroll
        for (int r = 0; r < RT; r++) {
          const float e = ex2(s[r] - (m_run[r] == -INFINITY ? 0.f : m_run[r]));
          l_run[r] += e;  // every quarter holds the same sum over its eight lanes
          if ((r & 3) == qd) sp[pp * RT + r] = e;
        }
        __syncwarp();
        const int np = min(8, rows - wr);
#pragma unroll
        for (int j = 0; j < 8; j += PS) {
          const int pos = j + (PS > 1 ? lane / CH : 0);
          if (pos < np) {
            float e[RT];
#pragma unroll
            for (int r = 0; r < RT; r++) e[r] = sp[pos * RT + r];
#pragma unroll
            for (int c = 0; c < NC; c++) {
              const float4 v = *reinterpret_cast<const float4*>(
                  vt + kv_at<TILE>(wr + pos, (lane % (CH < 32 ? CH : 32)) + 32 * c));
#pragma unroll
              for (int r = 0; r < RT; r++) {
                o[r][4 * c] += e[r] * v.x;
                o[r][4 * c + 1] += e[r] * v.y;
                o[r][4 * c + 2] += e[r] * v.z;
                o[r][4 * c + 3] += e[r] * v.w;
              }
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&ring->empty[sl.i]);
    }
#pragma unroll
    for (int r = 0; r < RT; r++) {
#pragma unroll
      for (int x = 1; x < 8; x <<= 1) l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], x);
      if constexpr (PS > 1) {
#pragma unroll
        for (int j = 0; j < NC * 4; j++) o[r][j] += __shfl_xor_sync(0xffffffffu, o[r][j], CH);
      }
    }
    consumer_sync<HS>(0);  // the last pair's states are read
    if (CH >= 32 || lane < CH) {
      const int col = (lane % (CH < 32 ? CH : 32)) * 4;
#pragma unroll
      for (int r = 0; r < RT; r++) {
        float* st = merge + (warp * RT + r) * kv_state_row<HS>();
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
          for (int e = 0; e < 4; e += 2)
            *reinterpret_cast<float2*>(st + 128 * c + col + e) = make_float2(o[r][4 * c + e], o[r][4 * c + e + 1]);
        if (lane == 0) {
          st[HS] = m_run[r];
          st[HS + 1] = l_run[r];
        }
      }
    }
    consumer_sync<HS>(0);
    kv_join<float, HS, RT>(p, merge, tid, w.seq, h0, 0, nh, w.tile == 0 && n == w.ntile, first ? 0 : 1);
  }
}

// Five to eight heads.  A lane owns one 16-byte chunk of every row (two at 256
// dimensions) of q, keys, values and output: q and the output stay in
// registers, and a key or value is read from shared memory once for all
// heads.  Rows of 64 dimensions have half as many chunks as the warp has
// lanes; its halves then share out the heads.  The products of four positions
// and four heads at a time are reduced over the lanes by halving; the scores
// go to the softmax through shared memory, two per lane of the same head
// throughout, and the weights come back as pairs (e, e) for packed
// multiplications.  Against the form above with eight heads, where q is read
// from shared memory for every position (64 requests, 4 kv heads, 524 MB): 8
// heads of 64 104 us (183), 12 of 64 184 (238), 8 of 256 108 (126), 8 of 128
// 102 (105); with four heads of 64, 128 and 256 it took 88, 86 and 93 us
// against 85, 86 and 87.  Bound by the issue of instructions.
template <int HS>
struct F32Lanes {
  static constexpr int kRow = HS < 128 ? HS / 4 : 32;  // lanes of a row
  static constexpr int kChunks = HS / 4 / kRow;        // chunks of a lane
  static constexpr int kHeads = kPaHeads * kRow / 32;  // heads of a lane
  // floats of a warp: scores [8][heads], weights [8][heads][2], rescales [heads][2]
  static_assert(26 <= kv_state_row<HS>(), "they lie where the warp's states will");
};

template <int HS, int SG>
VDEV void kv_consume_f32_wide(const KvAttnParams& p, KvWalk<kv_tile<float, HS>()> w, KvRing* ring, uint8_t* stages,
                         float* merge) {
  using FL = F32Lanes<HS>;
  constexpr int TILE = kv_tile<float, HS>(), NW = kv_warps<HS>(), RT = kPaHeads, LPR = FL::kRow, NC = FL::kChunks;
  constexpr int NH = FL::kHeads, HB = 4, PB = 4, NS = HB * PB, ROW = kv_state_row<HS>();
  static_assert(NS <= LPR, "a lane ends with one sum");
  const int lane = threadIdx.x & 31, cl = lane % LPR, hb0 = NH < RT ? lane / LPR * NH : 0;
  const int sg = SG == 1 ? 0 : (int)(threadIdx.x >> 5) / NW;  // the group, and the warp in it
  const int warp = (int)(threadIdx.x >> 5) - sg * NW;
  merge += sg * kv_merge_floats<float, HS, RT, 1>();
  float* sc = merge + warp * RT * ROW;  // scores
  float* we = sc + 8 * RT;              // weights
  float* al = we + 16 * RT;             // rescales
  const int wr = 8 * warp;
  const int sh = lane % RT, sp0 = lane / RT;  // softmax: this lane's head, and positions sp0 and sp0 + 4
  KvSlot sl;
  for (bool first = true; w.left > 0; w.next(p), first = false) {
    const int kh = w.kh, sub = w.sub, n = w.count();
    const int first_h = sub * p.heads + sg * kPaHeads, nh = min(RT, p.R - first_h), h0 = kh * p.R + first_h;
    f2 q[NH][NC][2], o[NH][NC][2];
    {
      const float* src = reinterpret_cast<const float*>(p.q) + (int64_t)w.seq * p.q_stride + (int64_t)h0 * HS;
#pragma unroll
      for (int r = 0; r < NH; r++)
#pragma unroll
        for (int c = 0; c < NC; c++) {
          q[r][c][0] = q[r][c][1] = o[r][c][0] = o[r][c][1] = f2_make(0.f, 0.f);
          if (hb0 + r < nh) load4(src + (hb0 + r) * HS + 4 * (cl + 32 * c), q[r][c]);
        }
    }
    prefetch_q<float, HS>(p, w);
    float m_run = -INFINITY, l_run = 0.f;  // of head sh, the sum over this lane's positions
    if (!first) consumer_sync<HS>(sg);     // the last pair's states are read
#pragma unroll 1
    for (int t = w.tile; t < w.tile + n; t++, sl.next()) {
      const bool ok = mbar_wait_lanes(&ring->full[sl.i], sl.phase, &ring->abort);
      if (!ok && lane == 0) {
        ring->abort = 1;
        set_error(p.err, VIREO_ERR_TIMEOUT);
      }
      const uint8_t* kt = stages + (size_t)sl.i * kv_stage_bytes<float, HS>();
      const uint8_t* vt = kt + TILE * HS * 4;
      const int rows = min(TILE, w.len - t * TILE);
      if (ok && wr < rows && nh > 0) {
#pragma unroll
        for (int j0 = 0; j0 < 8; j0 += PB) {
          f2 k[PB][NC][2];
#pragma unroll
          for (int j = 0; j < PB; j++)
#pragma unroll
            for (int c = 0; c < NC; c++)
              load4(reinterpret_cast<const float*>(kt + kv_at<TILE>(wr + j0 + j, cl + 32 * c)), k[j][c]);
#pragma unroll
          for (int r0 = 0; r0 < NH; r0 += HB) {
            float s[NS];
#pragma unroll
            for (int j = 0; j < PB; j++)
#pragma unroll
              for (int r = 0; r < HB; r++) {
                f2 d = f2_mul(q[r0 + r][0][0], k[j][0][0]);
                d = f2_fma(q[r0 + r][0][1], k[j][0][1], d);
#pragma unroll
                for (int c = 1; c < NC; c++) {
                  d = f2_fma(q[r0 + r][c][0], k[j][c][0], d);
                  d = f2_fma(q[r0 + r][c][1], k[j][c][1], d);
                }
                float x, y;
                f2_get(d, x, y);
                s[j * HB + r] = x + y;
              }
            // a lane whose bit is set keeps the upper half of the sums
#pragma unroll
            for (int b = NS / 2, by = LPR / 2; b >= 1; b >>= 1, by >>= 1) {
              const bool upper = (lane & by) != 0;
#pragma unroll
              for (int v = 0; v < b; v++) {
                const float send = upper ? s[v] : s[v + b], keep = upper ? s[v + b] : s[v];
                s[v] = keep + __shfl_xor_sync(0xffffffffu, send, by);
              }
            }
            if constexpr (LPR > NS) s[0] += __shfl_xor_sync(0xffffffffu, s[0], 1);
            const int v = cl / (LPR / NS);
            if (cl % (LPR / NS) == 0) sc[(j0 + v / HB) * RT + hb0 + r0 + v % HB] = s[0];
          }
        }
        __syncwarp();
        const float x0 = wr + sp0 < rows ? sc[sp0 * RT + sh] * p.scale : -INFINITY;
        const float x1 = wr + sp0 + 4 < rows ? sc[(sp0 + 4) * RT + sh] * p.scale : -INFINITY;
        float mt = fmaxf(x0, x1);
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 8));
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 16));
        const float m_new = fmaxf(m_run, mt), m_sub = m_new == -INFINITY ? 0.f : m_new;
        const bool up = __any_sync(0xffffffffu, m_new > m_run);
        if (up) {
          const float a = ex2(m_run - m_sub);
          l_run *= a;
          m_run = m_new;
          if (lane < RT) *reinterpret_cast<float2*>(al + 2 * lane) = make_float2(a, a);
        }
        const float e0 = ex2(x0 - m_sub), e1 = ex2(x1 - m_sub);
        l_run += e0 + e1;
        *reinterpret_cast<float2*>(we + 2 * (sp0 * RT + sh)) = make_float2(e0, e0);
        *reinterpret_cast<float2*>(we + 2 * ((sp0 + 4) * RT + sh)) = make_float2(e1, e1);
        __syncwarp();
        if (up) {
#pragma unroll
          for (int r = 0; r < NH; r++) {
            const f2 a = *reinterpret_cast<const f2*>(al + 2 * (hb0 + r));
#pragma unroll
            for (int c = 0; c < NC; c++) {
              o[r][c][0] = f2_mul(o[r][c][0], a);
              o[r][c][1] = f2_mul(o[r][c][1], a);
            }
          }
        }
        const int np = min(8, rows - wr);
#pragma unroll
        for (int pos = 0; pos < 8; pos++)
          if (pos < np) {
            f2 v[NC][2], e[NH];
#pragma unroll
            for (int c = 0; c < NC; c++)
              load4(reinterpret_cast<const float*>(vt + kv_at<TILE>(wr + pos, cl + 32 * c)), v[c]);
#pragma unroll
            for (int r = 0; r < NH; r += 2) load4(we + 2 * (pos * RT + hb0 + r), e + r);
#pragma unroll
            for (int r = 0; r < NH; r++)
#pragma unroll
              for (int c = 0; c < NC; c++) {
                o[r][c][0] = f2_fma(e[r], v[c][0], o[r][c][0]);
                o[r][c][1] = f2_fma(e[r], v[c][1], o[r][c][1]);
              }
          }
      }
      __syncwarp();  // also: the warp's scores and weights are read
      if (lane == 0) mbar_arrive(&ring->empty[sl.i]);
    }
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 8);
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 16);
    float* st = merge + warp * RT * ROW;
#pragma unroll
    for (int r = 0; r < NH; r++)
#pragma unroll
      for (int c = 0; c < NC; c++) {
        float v[4];
        f2_get(o[r][c][0], v[0], v[1]);
        f2_get(o[r][c][1], v[2], v[3]);
        float2* d = reinterpret_cast<float2*>(st + (hb0 + r) * ROW + 4 * (cl + 32 * c));
        d[0] = make_float2(v[0], v[1]);
        d[1] = make_float2(v[2], v[3]);
      }
    if (lane < RT) {
      st[lane * ROW + HS] = m_run;
      st[lane * ROW + HS + 1] = l_run;
    }
    consumer_sync<HS>(sg);
    kv_join<float, HS, RT>(p, merge, threadIdx.x - 32 * NW * sg, w.seq, h0, sg, nh, w.tile == 0 && n == w.ntile,
                           first ? 0 : 1);
  }
}

template <class TA, class TC, int HS, int RT, int SG, bool RUNS>
__global__ void __launch_bounds__(kv_threads<HS, SG>(), HS == 256 || SG == 2 ? 1 : 2)
    kv_attn_kernel(const __grid_constant__ KvAttnParams p, const __grid_constant__ CUtensorMap mk,
                   const __grid_constant__ CUtensorMap mv) {
  // stages first: the swizzle's atoms are 1024 bytes, and shared memory that
  // is all dynamic starts on such a boundary (checked below)
  extern __shared__ __align__(1024) uint8_t stages[];
  float* merge = reinterpret_cast<float*>(stages + kPaStages * kv_stage_bytes<TC, HS>());
  KvRing* ring = reinterpret_cast<KvRing*>(merge + kv_merge_floats<TC, HS, RT, SG>());
  if (threadIdx.x == 0) {
    for (int s = 0; s < kPaStages; s++) {
      mbar_init(&ring->full[s], 2);
      mbar_init(&ring->empty[s], kv_warps<HS>() * SG);
    }
    ring->abort = 0;
    mbar_fence_init();
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mk) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mv) : "memory");
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  asm volatile("fence.proxy.async;" ::: "memory");  // pool rows written by the kernels before this one
  constexpr int TILE = kv_tile<TC, HS>();
  const auto w = p.whole ? kv_pair<TILE>(p) : p.small ? kv_start<int, TILE, kv_threads<HS, SG>() / 32>(p, ring)
                                          : kv_start<long long, TILE, kv_threads<HS, SG>() / 32>(p, ring);
  if (w.left <= 0) {
    if (p.whole) {  // zeros for a request without positions; else the merge writes them
      const int nh = min(p.heads, p.R - w.sub * p.heads);
      TA* out = reinterpret_cast<TA*>(p.out) + (int64_t)w.seq * p.out_stride +
                (int64_t)(w.kh * p.R + w.sub * p.heads) * HS;
      const float z[4] = {0.f, 0.f, 0.f, 0.f};
      for (int i = threadIdx.x * 4; i < nh * HS; i += kv_threads<HS, SG>() * 4) store_f<4>(out + i, z);
    }
    return;
  }
  if (smem_addr(stages) & 1023u) {
    set_error(p.err, VIREO_ERR_UNSUPPORTED);
    return;
  }
  if (threadIdx.x >= 32 * kv_warps<HS>() * SG) {
    const bool values = threadIdx.x >= 32 * (kv_warps<HS>() * SG + 1);
    kv_produce<TC, HS>(p, values ? &mv : &mk, w, ring, stages + (values ? kv_stage_bytes<TC, HS>() / 2 : 0),
                       values ? p.where : nullptr);
  } else if constexpr (sizeof(TC) == 2) {
    kv_consume_mma<TA, TC, HS, SG, RUNS>(p, w, ring, stages, merge);
  } else if constexpr (RT == kPaHeads) {
    kv_consume_f32_wide<HS, SG>(p, w, ring, stages, merge);
  } else {
    static_assert(SG == 1, "one group");
    kv_consume_f32<HS, RT>(p, w, ring, stages, merge);
  }
}

// Joins the partial states of a (request, kv head, sub) that several CTAs
// share, and writes the zeros of requests without positions.  Nothing is read
// ahead of its wait: only that makes what any kernel before wrote visible.
// The attention kernel leaves where the states are, which a CTA would else
// find from all lengths (1.5 us a call).  A thread holds
// four dimensions of one head; the thread groups take the states in turn, a
// running (maximum, sum, accumulator) each with kMergeAhead states loaded at
// once, and are joined through shared memory in group order.  With few
// requests blockIdx.z spreads the heads.
constexpr int kMergeThreads = 256;
constexpr int kMergeAhead = 8;
template <class TA, int HS>
__global__ void __launch_bounds__(kMergeThreads) kv_merge_kernel(const __grid_constant__ KvAttnParams p) {
  constexpr int TPR = HS / 4, NG = kMergeThreads / TPR;  // threads per row, groups
  __shared__ float2 gml[NG];
  __shared__ float4 gacc[NG][TPR];
  const int seq = blockIdx.x, unit = blockIdx.y, tid = threadIdx.x;
  const int kh = unit / p.nsub, sub = unit - kh * p.nsub;
  const int nh = min(p.heads, p.R - sub * p.heads), h0 = kh * p.R + sub * p.heads;
  TA* out = reinterpret_cast<TA*>(p.out) + (int64_t)seq * p.out_stride + (int64_t)h0 * HS;
  const int col = (tid % TPR) * 4, grp = tid / TPR;
  pdl_wait();
  const int2 where = __ldcg(p.where + (int64_t)seq * p.G * p.nsub + unit);  // unset without positions
  if (kv_len_of(p, seq) == 0) {
    const float z[4] = {0.f, 0.f, 0.f, 0.f};
    for (int h = blockIdx.z + gridDim.z * grp; h < nh; h += gridDim.z * NG) store_f<4>(out + h * HS + col, z);
    return;
  }
  const int c0 = where.x >> 1, nc = where.y;
  // (out of the grid only where the attention gave up and reported it)
  if (c0 < 0 || nc < 1 || c0 >= p.ctas || nc > p.ctas - c0) return;
  // this CTA's heads are z, z + gridDim.z, ...; the last sub of a kv head may have fewer heads than gridDim.z
  const int hc = (int)blockIdx.z < nh ? (nh - (int)blockIdx.z + (int)gridDim.z - 1) / (int)gridDim.z : 0;
  if (nc == 1 || hc == 0) return;  // finished by the pair's only CTA, or none to do
  int gph = 1;  // thread groups per head, a power of two (hc >= 1 ends the loop)
  while (2 * gph * hc <= NG) gph *= 2;
  const int side = NG / gph, part = grp & (gph - 1);  // heads at a time
  for (int hb = 0; hb < hc; hb += side) {
    const int hi = hb + grp / gph, h = blockIdx.z + hi * gridDim.z;
    const auto state = [&](int i) {
      return p.part + ((size_t)(i ? 2 * (c0 + i) : where.x) * p.heads + h) * (HS + 4);
    };
    float M = -INFINITY, L = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    if (hi < hc)
      for (int i0 = part; i0 < nc; i0 += gph * kMergeAhead) {
        float4 v[kMergeAhead];
        float2 ml[kMergeAhead];
        float m = M;
#pragma unroll
        for (int j = 0; j < kMergeAhead; j++) {
          const int i = i0 + j * gph;
          v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
          ml[j] = make_float2(-INFINITY, 0.f);
          if (i < nc) {
            v[j] = __ldcg(reinterpret_cast<const float4*>(state(i) + col));
            ml[j] = __ldcg(reinterpret_cast<const float2*>(state(i) + HS));
          }
        }
#pragma unroll
        for (int j = 0; j < kMergeAhead; j++) m = fmaxf(m, ml[j].x);
        const float m_sub = m == -INFINITY ? 0.f : m, f0 = ex2(M - m_sub);
        L *= f0;
#pragma unroll
        for (int e = 0; e < 4; e++) acc[e] *= f0;
#pragma unroll
        for (int j = 0; j < kMergeAhead; j++) {
          const float f = ex2(ml[j].x - m_sub);
          L += ml[j].y * f;
          acc[0] += v[j].x * f;
          acc[1] += v[j].y * f;
          acc[2] += v[j].z * f;
          acc[3] += v[j].w * f;
        }
        M = m;
      }
    gacc[grp][tid % TPR] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    if (col == 0) gml[grp] = make_float2(M, L);
    __syncthreads();
    if (part == 0 && hi < hc) {
      float m = -INFINITY;
      for (int g = grp; g < grp + gph; g++) m = fmaxf(m, gml[g].x);
      const float m_sub = m == -INFINITY ? 0.f : m;
      float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
      for (int g = grp; g < grp + gph; g++) {
        const float f = ex2(gml[g].x - m_sub);
        const float4 v4 = gacc[g][tid % TPR];
        l += gml[g].y * f;
        o[0] += v4.x * f;
        o[1] += v4.y * f;
        o[2] += v4.z * f;
        o[3] += v4.w * f;
      }
      const float f = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);  // a NaN stays one
#pragma unroll
      for (int e = 0; e < 4; e++) o[e] *= f;
      store_f<4>(out + h * HS + col, o);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Block selection.
//
// kv_score_kernel: a warp takes eight pages and eight of the kv head's q heads
// (two times eight where there are more) and multiplies them with 64-bit
// matrix instructions.  Products of a 16-bit or fp32 key with an fp32 query
// are exact in 64 bits; each addition rounds, so a score is off by at most
// head_size * 2^-53 of the sum of its products' magnitudes, and only pages
// closer than that (not those of equal means, which take the same steps)
// depend on the order of the additions.  A key element is converted by
// one lane, once; a lane group per page with its sums reduced over the lanes
// spent its time on conversions repeated for the heads and on shuffles (8
// requests up to 109k positions, 4 x 12 heads of 64, pages of 32: 40 us
// against 12).  The maximum over heads becomes a sortable 64-bit key.  Bound by
// latency (length, page number, key, one after the other) and, for many
// pages, by the 64-bit rate.
// kv_select_kernel: one CTA per (request, kv head) finds the n_top-th
// largest key.  A histogram of 256 bins, for a small n_top over the two
// octaves below the largest score, leaves a few keys in question, which are
// ranked against one another; where it leaves more than kSelList, a histogram
// over those follows (9 requests, 800 candidates, 4 kv heads: 22.6 us in all
// against 25.5 with histograms of the eight bits below those that all share).
// The chosen pages are written in rising order, as indices and as pool
// pages.  Bound by the latency of its steps (barriers, scans): as
// few warps as keep the candidates in registers, eight each, up to 8192 of
// them (3 requests, 2500 candidates: 17.6 us in all with 16 warps, 21.5 with
// 32; 6500 candidates, 18 pairs: 68 us with eight warps that read them again
// for every step).
// ---------------------------------------------------------------------------
struct KvSelectParams {
  const void* q;
  const void* means;
  int64_t q_stride, table_stride;
  const int32_t *table, *kv_len;
  int max_pages, n_pages, H, G, R, ps_shift, n_sink, n_window, n_top, nsel;
  uint64_t* keys;  // [n_seqs][G][max_pages]
  int32_t* phys;   // [n_seqs][G][nsel]
  int32_t* sel;    // the caller's, or null
  int* err;
};

VDEV int select_pages(const KvSelectParams& p, int seq) {
  const int n = min(max(p.kv_len[seq], 0), p.max_pages << p.ps_shift);
  return (n + (1 << p.ps_shift) - 1) >> p.ps_shift;
}

// order of doubles as unsigned integers; NaN below everything, -0 as +0
VDEV uint64_t sort_key(double v) {
  if (isnan(v)) return 0ull;
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
  return b & (1ull << 63) ? ~b : b | (1ull << 63);
}

constexpr int kScoreThreads = 128;
constexpr int kScorePages = 8;  // of a warp

// c[8 heads][8 pages] += a[8 heads][4 dimensions] b[4 dimensions][8 pages], in 64 bits
VDEV void mma_f64(double (&c)[2], double a, double b) {
  asm("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};"
      : "+d"(c[0]), "+d"(c[1])
      : "d"(a), "d"(b));
}

template <class TA, class TC, int HS, int RB>
__global__ void __launch_bounds__(kScoreThreads) kv_score_kernel(const __grid_constant__ KvSelectParams p, int per) {
  // four lanes to a page, 16 bytes (E values) of every 64 to a lane; HS / 4
  // steps of four dimensions, the lanes' e-th of their i-th load each
  constexpr int E = 16 / (int)sizeof(TC), NL = HS / (4 * E), NP = kScorePages;
  __shared__ double qs[RB][HS / 4][33];  // a step's lanes side by side; 33: the stores meet fewer conflicts
  pdl_wait();
  pdl_launch_dependents();
  const int seq = blockIdx.z, g = blockIdx.y;
  const int np = select_pages(p, seq);
  if (np <= p.nsel) return;
  const int lo = p.n_sink + blockIdx.x * per, hi = min(np - p.n_window, lo + per);
  if (lo >= hi) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = lane & 3;
  const int32_t* row = p.table + (int64_t)seq * p.table_stride;
  const TC* means = (const TC*)p.means + g * HS + c * E;
  uint64_t* keys = p.keys + ((int64_t)seq * p.G + g) * p.max_pages;
  // page numbers of the warp's pages from base on, lane by lane
  const auto numbers = [&](int base) { return lane < NP && base + lane < hi ? row[base + lane] : -1; };
  const auto checked = [&](int base, int id) {  // a page outside the pool: zeros
    if (id >= 0 && id < p.n_pages) return id;
    if (lane < NP && base + lane < hi) set_error(p.err, VIREO_ERR_ARG);
    return -1;
  };
  const auto load = [&](const TC* src, int i) {
    return src ? *reinterpret_cast<const uint4*>(src + 4 * E * i) : make_uint4(0u, 0u, 0u, 0u);
  };
  for (int r0 = 0; r0 < p.R; r0 += 8 * RB) {
    int base = lo + warp * NP;
    const int step = kScoreThreads / 32 * NP;
    int ahead = numbers(base);
    const TA* q = (const TA*)p.q + (int64_t)seq * p.q_stride + (int64_t)(g * p.R + r0) * HS;
    const int nq = min(8 * RB, p.R - r0) * HS;
    if (r0) __syncthreads();  // the last heads' are read
#pragma unroll 4
    for (int i = threadIdx.x; i < 8 * RB * HS; i += kScoreThreads) {
      const int h = i / HS, d = i % HS, v = d / E;  // vector v is lane v % 4's (v / 4)-th
      qs[h / 8][v / 4 * E + d % E][(h % 8) * 4 + (v & 3)] = i < nq ? (double)to_f(q[i]) : 0.0;
    }
    const auto point = [&](int id) {
      const int pg = __shfl_sync(0xffffffffu, id, lane >> 2);
      return pg >= 0 ? means + (int64_t)pg * p.G * HS : nullptr;
    };
    uint4 k[NL];  // as loaded, the next page's in place of each that has been used
    const TC* src = point(checked(base, ahead));
#pragma unroll
    for (int i = 0; i < NL; i++) k[i] = load(src, i);
    ahead = numbers(base + step);
    __syncthreads();
    for (; base < hi; base += step) {
      src = point(checked(base + step, ahead));
      ahead = numbers(base + 2 * step);
      double s[RB][2];
#pragma unroll
      for (int b = 0; b < RB; b++) s[b][0] = s[b][1] = 0.0;
#pragma unroll
      for (int i = 0; i < NL; i++) {
#pragma unroll
        for (int e = 0; e < E; e++) {
          const double kd = (double)to_f(reinterpret_cast<const TC*>(&k[i])[e]);
#pragma unroll
          for (int b = 0; b < RB; b++) mma_f64(s[b], qs[b][i * E + e][lane], kd);
        }
        k[i] = load(src, i);
      }
      // lane 4 h + c has head h's scores of pages 2 c and 2 c + 1
#pragma unroll
      for (int j = 0; j < 2; j++) {
        uint64_t key = 0;
#pragma unroll
        for (int b = 0; b < RB; b++) {
          const uint64_t v = r0 + 8 * b + (lane >> 2) < p.R ? sort_key(s[b][j]) : 0ull;
          key = v > key ? v : key;
        }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          const uint64_t other = __shfl_xor_sync(0xffffffffu, key, o);
          key = other > key ? other : key;
        }
        const int pg = base + 2 * c + j;
        if (lane < 4 && pg < hi) keys[pg] = r0 ? max(key, keys[pg]) : key;
      }
    }
  }
}

constexpr int kSelBits = 8, kSelBins = 1 << kSelBits;  // a thread per bin
constexpr int kSelNear = 53 - kSelBits;                // 2^53: two octaves of doubles
constexpr int kSelList = 256;                          // candidates ranked directly
constexpr int kSelKeep = 8;                            // keys a thread keeps in registers

template <int kSelThreads>
__global__ void __launch_bounds__(kSelThreads) kv_select_kernel(const __grid_constant__ KvSelectParams p) {
  constexpr int kSelWarps = kSelThreads / 32;
  static_assert(kSelThreads >= kSelBins && kSelThreads >= kSelList, "a thread per bin and per candidate");
  __shared__ unsigned int hist[kSelBins];
  __shared__ uint64_t list[kSelList];
  __shared__ uint64_t top[kSelWarps];
  __shared__ int wsum[2][kSelWarps];
  __shared__ int pick[3];
  __shared__ unsigned int n_list;
  __shared__ uint64_t t_key;
  __shared__ int t_eq;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < kSelBins) hist[tid] = 0;
  if (tid == 0) n_list = 0;
  pdl_wait();
  pdl_launch_dependents();
  const int seq = blockIdx.y, g = blockIdx.x;
  const int np = select_pages(p, seq), ns = min(np, p.nsel);
  const int32_t* row = p.table + (int64_t)seq * p.table_stride;
  int32_t* phys = p.phys + ((int64_t)seq * p.G + g) * p.nsel;
  int32_t* sel = p.sel ? p.sel + ((int64_t)seq * p.G + g) * p.nsel : nullptr;
  const auto put = [&](int at, int page) {
    phys[at] = row[page];
    if (sel) sel[at] = page;
  };
  if (sel)
    for (int i = ns + tid; i < p.nsel; i += kSelThreads) sel[i] = -1;
  if (np <= p.nsel) {
    for (int i = tid; i < np; i += kSelThreads) put(i, i);
    return;
  }
  const int m = np - p.n_sink - p.n_window;  // candidates, more than n_top
  const uint64_t* keys = p.keys + ((int64_t)seq * p.G + g) * p.max_pages + p.n_sink;
  // a thread's run of neighbouring keys
  const int run = (m + kSelThreads - 1) / kSelThreads, i0 = min(m, tid * run), i1 = min(m, i0 + run);
  const bool keep = run <= kSelKeep;
  uint64_t mine[kSelKeep];
  if (keep && p.n_top)
#pragma unroll
    for (int j = 0; j < kSelKeep; j++) mine[j] = i0 + j < i1 ? __ldcg(keys + i0 + j) : 0ull;
  const auto each = [&](auto&& f) {
    if (keep) {
#pragma unroll
      for (int j = 0; j < kSelKeep; j++)
        if (i0 + j < i1) f(i0 + j, mine[j]);
    } else {
      for (int i = i0; i < i1; i++) f(i, __ldcg(keys + i));
    }
  };
  // the same in any order
  const auto some = [&](auto&& f) {
    if (keep) {
      each(f);
    } else {
#pragma unroll 4
      for (int i = tid; i < m; i += kSelThreads) f(i, __ldcg(keys + i));
    }
  };
  for (int i = tid; i < p.n_sink; i += kSelThreads) put(i, i);
  for (int i = tid; i < p.n_window; i += kSelThreads) put(p.n_sink + p.n_top + i, np - p.n_window + i);
  if (p.n_top == 0) return;

  // the largest key
  uint64_t hi = 0;
  some([&](int, uint64_t k) { hi = max(hi, k); });
#pragma unroll
  for (int o = 16; o; o >>= 1) hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  if (lane == 0) top[warp] = hi;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSelWarps; w++) hi = max(hi, top[w]);
  // Keys of [lo, hi] are in question, `equal` of them, of which the `want`
  // largest are to be taken.  Where a small part is, the first 255 bins are
  // spread over two octaves below the largest score and the last has the
  // rest; else, and from then on, they cover all that is in question.
  uint64_t lo = 0;
  int want = p.n_top, equal = m;
  bool near = (int64_t)p.n_top * 6 < m;
  const auto asked = [&](uint64_t k) { return k >= lo && k <= hi; };
  while (equal > kSelList && hi > lo) {
    const int s = near ? kSelNear : max(0, 64 - kSelBits - __clzll((long long)(hi - lo)));
    some([&](int, uint64_t k) {
      if (asked(k)) atomicAdd(&hist[min((unsigned int)min((hi - k) >> s, (uint64_t)kSelBins), kSelBins - 1u)], 1u);
    });
    __syncthreads();
    const int c = tid < kSelBins ? (int)hist[tid] : 0;  // bin 0 is the top one
    int inc = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    if (lane == 31) wsum[0][warp] = inc;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSelWarps; w++) inc += w < warp ? wsum[0][w] : 0;
    if (tid < kSelBins) hist[tid] = 0;  // every bin has been read
    if (c && inc - c < want && inc >= want) {  // one thread
      pick[0] = tid;
      pick[1] = inc - c;
      pick[2] = c;
    }
    __syncthreads();
    const uint64_t span = (1ull << s) - 1;
    hi -= (uint64_t)pick[0] << s;
    if (!(near && pick[0] == kSelBins - 1) && hi > span) lo = max(lo, hi - span);
    want -= pick[1];
    equal = pick[2];
    near = false;
  }
  // The smallest key to be taken and how many of its equals: by rank among
  // those in question, or, where more than kSelList are all alike, the key
  // itself with `want` of them.
  uint64_t tk = hi;
  int teq = want;
  if (equal <= kSelList) {
    some([&](int, uint64_t k) {
      if (asked(k)) list[atomicAdd(&n_list, 1u)] = k;
    });
    __syncthreads();
    if (tid < equal) {
      const uint64_t k = list[tid];
      int above = 0, same = 0;
      for (int j = 0; j < equal; j++) {
        const uint64_t o = list[j];
        above += o > k;
        same += o == k;
      }
      if (above < want && above + same >= want) {  // several threads with the same values
        t_key = k;
        t_eq = want - above;
      }
    }
    __syncthreads();
    tk = t_key;
    teq = t_eq;
  }
  // Taken: keys above tk, and the first teq at it, which are those of the
  // lowest pages.  The runs' counts are scanned once.
  int more = 0, eq = 0;
  each([&](int, uint64_t k) {
    more += k > tk;
    eq += k == tk;
  });
  int smore = more, seq_ = eq;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, smore, o), v = __shfl_up_sync(0xffffffffu, seq_, o);
    if (lane >= o) {
      smore += u;
      seq_ += v;
    }
  }
  __syncthreads();  // wsum has been read
  if (lane == 31) {
    wsum[0][warp] = smore;
    wsum[1][warp] = seq_;
  }
  __syncthreads();
  int nh = smore - more, ne = seq_ - eq;  // above and at tk before this run
#pragma unroll
  for (int w = 0; w < kSelWarps; w++) {
    nh += w < warp ? wsum[0][w] : 0;
    ne += w < warp ? wsum[1][w] : 0;
  }
  if (more || (eq && ne < teq))
    each([&](int i, uint64_t k) {
      if (k > tk || (k == tk && ne < teq)) put(p.n_sink + nh + min(ne, teq), p.n_sink + i);
      nh += k > tk;
      ne += k == tk;
    });
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

static int kv_tile_of(const gguf_kv_desc& d) {
  const bool f32 = d.kv_type == KV_F32;
  if (d.head_size == 64) return f32 ? kv_tile<float, 64>() : kv_tile<__half, 64>();
  return f32 ? kv_tile<float, 128>() : kv_tile<__half, 128>();  // as at 256
}

// Pairs of at most this many tiles are not cut, each is a CTA's own: one launch
// instead of two.  Tiles by the table's width, which the host knows: a short
// request in a wide table is cut (one of 300 positions, 16 heads, 5.6 us in a
// table for 300, 6.9 in one for 32k).  A tile takes a CTA
// 0.5 to 1.7 us, the cut and the join about 3, and the second launch the host
// about 3.  One request, replayed, whole against cut: 32 / 4 heads of 128
// over a 16-bit cache, 4 tiles 5.1 / 6.2 us, 6 6.4 / 6.2, 8 7.6 / 6.3 (eight
// such requests 5.2 / 7.8, 6.5 / 8.3, 7.7 / 8.6); 32 / 4 of 256 4 tiles 7.0 /
// 7.4, 6 8.8 / 7.5; 48 / 4 of 128 6 tiles 7.2 / 6.6; an fp32 cache, 16 / 16 of
// 128 8 tiles 6.4 / 5.7, 16 / 4 4 tiles 6.2 / 6.1, 32 / 4 4 tiles 7.6 / 6.5,
// 16 / 2 of 256 2 tiles 6.3 / 7.4, 4 9.7 / 7.4.  With pairs for more than half
// of the CTAs that the GPU holds the cut brings less and the limit is twice
// that, with pairs for more than all of them four times (ragged requests, 32 /
// 4 of 128, bf16: 40 of up to 1024 positions, 16 tiles, 13.6 / 14.9 us, of up
// to 2048 23.6 / 18.8; 128 requests 29.7 / 35.6 and 52.6 / 53.4; 256 requests
// 51.4 / 59.6 and 92.6 / 96.2), up to four times as many pairs as that (41
// requests of 16 kv heads, one position each: 11.0 / 15.2; 512 of 8: 48 / 46).
template <class TC, int HS, int RT, int SG>
constexpr int kv_whole_tiles() {
  return sizeof(TC) == 4 ? (RT == 8 ? 4 : RT == 4 ? 5 : 8) - (HS == 256) : HS == 256 ? 5 : SG == 2 ? 6 : 8;
}

constexpr int kPaWholeWaves = 4;
static_assert(4 * kv_whole_tiles<__half, 64, kPaHeads, 1>() <= kPaRun, "a whole pair is one run");

struct KvKernel {
  const void *fn, *runs;  // runs: for more than kPaRun tiles of a pair in a CTA
  int smem, threads, heads, whole_tiles;
};
template <class TA, class TC, int HS, int RT, int SG = 1>
static KvKernel kv_kernel() {
  static_assert(kv_attn_smem<TC, HS, RT, SG>() <= 227 * 1024, "the most shared memory a CTA can have");
  return {reinterpret_cast<const void*>(&kv_attn_kernel<TA, TC, HS, RT, SG, false>),
          reinterpret_cast<const void*>(&kv_attn_kernel<TA, TC, HS, RT, SG, sizeof(TC) == 2>),
          kv_attn_smem<TC, HS, RT, SG>(), kv_threads<HS, SG>(), SG * kPaHeads, kv_whole_tiles<TC, HS, RT, SG>()};
}
template <class TA, class TC>
static KvKernel kv_kernel_h(int hs, int R) {
  switch (hs) {
    case 64: return R > kPaHeads ? kv_kernel<TA, TC, 64, kPaHeads, 2>() : kv_kernel<TA, TC, 64, kPaHeads>();
    case 128: return R > kPaHeads ? kv_kernel<TA, TC, 128, kPaHeads, 2>() : kv_kernel<TA, TC, 128, kPaHeads>();
    default: return kv_kernel<TA, TC, 256, kPaHeads>();
  }
}
// fp32 cache: the smallest of 1, 2, 4, 8 heads that holds the group
template <int HS>
static KvKernel kv_kernel_f32(int R) {
  if (R == 1) return kv_kernel<float, float, HS, 1>();
  if (R == 2) return kv_kernel<float, float, HS, 2>();
  if (R <= 4) return kv_kernel<float, float, HS, 4>();
  if constexpr (HS < 256)
    if (R > kPaHeads) return kv_kernel<float, float, HS, 8, 2>();
  return kv_kernel<float, float, HS, 8>();
}
static KvKernel kv_kernel_for(const gguf_kv_desc& d) {
  const int R = d.n_heads / d.n_kv_heads;
  if (d.act_type == KV_BF16) return kv_kernel_h<__nv_bfloat16, __nv_bfloat16>(d.head_size, R);
  if (d.act_type == KV_F16) return kv_kernel_h<__half, __half>(d.head_size, R);
  if (d.kv_type == KV_F16) return kv_kernel_h<float, __half>(d.head_size, R);
  return d.head_size == 64 ? kv_kernel_f32<64>(R) : d.head_size == 128 ? kv_kernel_f32<128>(R) : kv_kernel_f32<256>(R);
}

template <class TA>
static const void* kv_merge_h(int hs) {
  switch (hs) {
    case 64: return reinterpret_cast<const void*>(&kv_merge_kernel<TA, 64>);
    case 128: return reinterpret_cast<const void*>(&kv_merge_kernel<TA, 128>);
    default: return reinterpret_cast<const void*>(&kv_merge_kernel<TA, 256>);
  }
}
static const void* kv_merge_for(const gguf_kv_desc& d) {
  if (d.act_type == KV_BF16) return kv_merge_h<__nv_bfloat16>(d.head_size);
  return d.act_type == KV_F16 ? kv_merge_h<__half>(d.head_size) : kv_merge_h<float>(d.head_size);
}

// CTAs of the attention kernel that the workspace has room for: two to an SM
// of up to 256 SMs; the launch takes as many as are resident
constexpr int kPaMaxCtas = 512;

template <class TA, class TC, int HS>
static const void* score_kernel(int R) {
  return R > 8 ? reinterpret_cast<const void*>(&kv_score_kernel<TA, TC, HS, 2>)
               : reinterpret_cast<const void*>(&kv_score_kernel<TA, TC, HS, 1>);
}
template <class TA, class TC>
static const void* score_kernel_h(int hs, int R) {
  switch (hs) {
    case 64: return score_kernel<TA, TC, 64>(R);
    case 128: return score_kernel<TA, TC, 128>(R);
    default: return score_kernel<TA, TC, 256>(R);
  }
}
static const void* score_kernel_for(const gguf_kv_desc& d) {
  const int R = d.n_heads / d.n_kv_heads;
  if (d.act_type == KV_BF16) return score_kernel_h<__nv_bfloat16, __nv_bfloat16>(d.head_size, R);
  if (d.act_type == KV_F16) return score_kernel_h<__half, __half>(d.head_size, R);
  if (d.kv_type == KV_F16) return score_kernel_h<float, __half>(d.head_size, R);
  return score_kernel_h<float, float>(d.head_size, R);
}

static size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }
// the workspace: partial states and where each pair's are, then with block
// selection scores and pages
struct KvWs {
  size_t part, where, keys, phys, total;
};
static KvWs kv_ws(const gguf_kv_desc& d, int n_seqs, int max_pages, int nsel) {
  KvWs w;
  w.part = 0;
  w.where = up256((size_t)kPaMaxCtas * 2 * kPaHeads * (d.head_size + 4) * 4);
  const size_t subs = (d.n_heads / d.n_kv_heads + kPaHeads - 1) / kPaHeads;  // at most
  w.keys = w.where + up256((size_t)n_seqs * d.n_kv_heads * subs * sizeof(int2));
  w.phys = w.keys + (nsel ? up256((size_t)n_seqs * d.n_kv_heads * max_pages * 8) : 0);
  w.total = w.phys + (nsel ? up256((size_t)n_seqs * d.n_kv_heads * nsel * 4) : 0);
  return w;
}

static int kv_attn_launch(gguf_kv* kv, const gguf_kv_attn_args& a, const int32_t* phys, int nsel, Ctx* c,
                          cudaStream_t s) {
  const gguf_kv_desc& d = kv->d;
  int st;
  const KvKernel k = kv_kernel_for(d);
  CUtensorMap mk, mv;
  int per_sm = 0;
  {
    std::lock_guard<std::mutex> lk(kv->mu);
    if (!kv->maps_ok) {
      if ((st = kv_make_map(d, kv_tile_of(d), &kv->map_k, d.k)) || (st = kv_make_map(d, kv_tile_of(d), &kv->map_v, d.v))) return st;
      int per = INT_MAX;
      for (const void* fn : {k.fn, k.runs}) {
        int n = 0;
        if ((st = cuda_status(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, k.smem))) ||
            (st = cuda_status(cudaFuncSetAttribute(fn, cudaFuncAttributePreferredSharedMemoryCarveout,
                                                   cudaSharedmemCarveoutMaxShared))) ||
            (st = cuda_status(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, fn, k.threads, k.smem))))
          return st;
        per = std::min(per, n);
      }
      if (per < 1) return VIREO_ERR_UNSUPPORTED;
      kv->per_sm = per;
      kv->maps_ok = true;
    }
    mk = kv->map_k;
    mv = kv->map_v;
    per_sm = kv->per_sm;
  }
  KvAttnParams p;
  p.q = a.q;
  p.out = a.out;
  p.q_stride = a.q_stride;
  p.out_stride = a.out_stride;
  p.table = nsel ? phys : a.table;
  p.table_stride = a.table_stride;
  p.kv_len = a.kv_len;
  p.n_seqs = a.n_seqs;
  p.max_pages = a.max_pages;
  p.n_pages = d.n_pages;
  p.H = d.n_heads;
  p.G = d.n_kv_heads;
  p.R = d.n_heads / d.n_kv_heads;
  p.heads = k.heads;
  p.nsub = (p.R + p.heads - 1) / p.heads;
  p.ps_shift = kv->ps_shift;
  p.nsel = nsel;
  p.scale = (a.scale == 0.f ? 1.0f / sqrtf((float)d.head_size) : a.scale) * kLog2e;
  p.part = (float*)a.ws;
  p.err = c->d_err;
  // no more CTAs than tiles there can be
  const int tile = kv_tile_of(d);
  const int64_t most = (int64_t)a.n_seqs * p.G * p.nsub *
                       (((int64_t)(nsel ? std::min(nsel, a.max_pages) : a.max_pages) * d.page_size + tile - 1) / tile);
  p.ctas = (int)std::min<int64_t>(std::min(kPaMaxCtas * kPaHeads / p.heads, c->num_sms * per_sm), most);
  p.sms = c->num_sms;
  const int64_t pairs = (int64_t)a.n_seqs * p.G * p.nsub;
  const int64_t held = (int64_t)c->num_sms * per_sm;
  p.whole = pairs <= kPaWholeWaves * held &&
            most <= pairs * k.whole_tiles * (pairs > held ? 4 : 2 * pairs > held ? 2 : 1);
  if (p.whole) p.ctas = (int)pairs;
  p.where = p.whole ? nullptr : (int2*)((uint8_t*)a.ws + kv_ws(d, a.n_seqs, a.max_pages, 0).where);
  p.small = most <= INT32_MAX;
  // the longest stretch of a CTA: `cut_ctas` takes fewer than p.ctas only for short lines
  const int64_t wide = (most + p.ctas - 1) / p.ctas, narrow = (kPaStages * (int64_t)p.ctas + p.sms - 1) / p.sms;
  const void* fn = !p.whole && std::max(wide, narrow) > kPaRun ? k.runs : k.fn;
  void* args[] = {&p, &mk, &mv};
  if ((st = launch_pdl_c(fn, dim3(p.ctas), dim3(k.threads), k.smem, s, args))) return st;
  if (p.whole) return VIREO_OK;
  // heads over CTAs while the pairs alone leave SMs idle
  const int hz = (int)std::min<int64_t>(std::min(p.R, p.heads), std::max<int64_t>(1, 2 * c->num_sms / pairs));
  return launch_pdl_c(kv_merge_for(d), dim3(a.n_seqs, p.G * p.nsub, hz), dim3(kMergeThreads), 0, s, args);
}

}  // namespace vireo

using namespace vireo;

extern "C" {

size_t gguf_kv_workspace(const gguf_kv* kv, int n_seqs, int max_pages, int n_select) {
  if (!kv || n_seqs < 0 || max_pages < 1 || n_select < 0) return 0;
  return kv_ws(kv->d, n_seqs, max_pages, n_select).total;
}

int gguf_kv_attn(gguf_kv* kv, const gguf_kv_attn_args* a, void* stream) {
  int st = kv_attn_check(kv, a);
  if (st) return st;
  if (a->n_seqs == 0) return VIREO_OK;
  if (a->ws_bytes < kv_ws(kv->d, a->n_seqs, a->max_pages, 0).total) return VIREO_ERR_ARG;
  Ctx* c = ctx_get(&st);
  if (!c) return st;
  DeviceGuard dg(c->device);
  if (dg.status) return dg.status;
  return kv_attn_launch(kv, *a, nullptr, 0, c, stream ? (cudaStream_t)stream : c->stream);
}

int gguf_kv_attn_topk(gguf_kv* kv, const gguf_kv_attn_args* a, const gguf_kv_select_args* sa, void* stream) {
  int st = kv_attn_check(kv, a);
  if (st) return st;
  if (!sa || sa->n_sink < 0 || sa->n_window < 1 || sa->n_top < 0 ||
      (int64_t)sa->n_sink + sa->n_window + sa->n_top > INT32_MAX / 1024)
    return VIREO_ERR_ARG;
  if (a->n_seqs == 0) return VIREO_OK;
  if (!sa->means || !kv_aligned(sa->means, 16)) return VIREO_ERR_ARG;
  const gguf_kv_desc& d = kv->d;
  const int nsel = sa->n_sink + sa->n_window + sa->n_top;
  const KvWs w = kv_ws(d, a->n_seqs, a->max_pages, nsel);
  if (a->ws_bytes < w.total) return VIREO_ERR_ARG;
  if (a->n_seqs > 65535 || d.n_kv_heads > 65535) return VIREO_ERR_UNSUPPORTED;
  Ctx* c = ctx_get(&st);
  if (!c) return st;
  DeviceGuard dg(c->device);
  if (dg.status) return dg.status;
  cudaStream_t s = stream ? (cudaStream_t)stream : c->stream;
  KvSelectParams p;
  p.q = a->q;
  p.means = sa->means;
  p.q_stride = a->q_stride;
  p.table = a->table;
  p.table_stride = a->table_stride;
  p.kv_len = a->kv_len;
  p.max_pages = a->max_pages;
  p.n_pages = d.n_pages;
  p.H = d.n_heads;
  p.G = d.n_kv_heads;
  p.R = d.n_heads / d.n_kv_heads;
  p.ps_shift = kv->ps_shift;
  p.n_sink = sa->n_sink;
  p.n_window = sa->n_window;
  p.n_top = sa->n_top;
  p.nsel = nsel;
  p.keys = (uint64_t*)((uint8_t*)a->ws + w.keys);
  p.phys = (int32_t*)((uint8_t*)a->ws + w.phys);
  p.sel = sa->sel;
  p.err = c->d_err;
  const int cand = a->max_pages - sa->n_sink - sa->n_window;
  if (a->max_pages > nsel && sa->n_top > 0) {
    // Pages per CTA: what its warps take at once, or as many times that as
    // leave eight CTAs per SM for requests as long as the table (most are
    // shorter).  16 requests up to 32k positions, the whole call, with 2, 4, 8
    // and 16 CTAs per SM: 31.0, 27.5, 26.5 and 26.6 us; 8 requests up to 109k:
    // 44.3, 41.6, 40.7 and 41.2.
    const int unit = kScoreThreads / 32 * kScorePages;
    const int64_t units = (int64_t)a->n_seqs * d.n_kv_heads * ((cand + unit - 1) / unit);
    int per = unit * (int)std::max<int64_t>(1, units / ((int64_t)c->num_sms * 8));
    void* args[] = {&p, &per};
    if ((st = launch_pdl_c(score_kernel_for(d), dim3((cand + per - 1) / per, d.n_kv_heads, a->n_seqs),
                           dim3(kScoreThreads), 0, s, args)))
      return st;
  }
  void* sargs[] = {&p};
  // the fewest threads that keep the candidates in registers, of 256, 512 and 1024
  const void* sel_fn = reinterpret_cast<const void*>(&kv_select_kernel<256>);
  int threads = 256;
  if (cand > 512 * kSelKeep) {
    sel_fn = reinterpret_cast<const void*>(&kv_select_kernel<1024>);
    threads = 1024;
  } else if (cand > 256 * kSelKeep) {
    sel_fn = reinterpret_cast<const void*>(&kv_select_kernel<512>);
    threads = 512;
  }
  if ((st = launch_pdl_c(sel_fn, dim3(d.n_kv_heads, a->n_seqs), dim3(threads), 0, s, sargs))) return st;
  return kv_attn_launch(kv, *a, p.phys, nsel, c, s);
}

}  // extern "C"
