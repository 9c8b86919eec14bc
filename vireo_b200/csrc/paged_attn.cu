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
//  * The copies never wait for the arithmetic: a producer warp walks the
//    tiles with TMA (a 4-D tensor map per pool: dimension, position, head,
//    page; one box per page and 128 bytes of a row, 128-byte swizzle) into a
//    ring of stages.  A page number outside the pool is out of the map's
//    bounds and reads as zeros.
//  * The arithmetic is small enough for mma.sync: up to eight q heads of a kv
//    head are the rows 0-7 of the M side.  Rows 8-15 would be empty; they hold
//    what rounding to the cache's type lost (of q where it is fp32, of the
//    softmax weights always), so both products keep about twice the type's
//    digits at no further instruction, and the two halves are added in fp32.
//    An fp32 cache runs on the CUDA cores in plain fp32.
//
// Softmax weights are exp2 of scores scaled by log2(e), with the running
// maximum and sum in fp32.
#include <math.h>

#include "paged_kv.cuh"
#include "pdl_launch.cuh"

namespace vireo {

constexpr int kPaWarps = 4;                      // consumer warps
constexpr int kPaThreads = 32 * (kPaWarps + 1);  // and one producer
constexpr int kPaConsumers = 32 * kPaWarps;
constexpr int kPaHeads = 8;                      // q heads a unit takes
constexpr int kPaStages = 3;
constexpr float kLog2e = 1.4426950408889634f;

// positions of a tile: what a stage of 16 or 32 KB of keys holds
template <class TC>
__host__ __device__ constexpr int kv_tile() { return sizeof(TC) == 4 ? 32 : 64; }
template <class TC, int HS>
__host__ __device__ constexpr int kv_stage_bytes() { return 2 * kv_tile<TC>() * HS * (int)sizeof(TC); }

struct KvAttnParams {
  const void* q;
  void* out;
  int64_t q_stride, out_stride, table_stride;
  const int32_t* table;  // block tables, or with nsel the chosen pages [n_seqs][G][nsel], physical
  const int32_t* kv_len;
  int n_seqs, max_pages, n_pages;
  int H, G, R, nsub;     // q heads, kv heads, heads per kv head, units per kv head
  int ps_shift, nsel, ctas;
  float scale;           // times log2(e)
  float* part;           // [ctas][2][kPaHeads][HS + 2]
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

// The line of tiles cut over the CTAs: units of request seq start at
// (tiles of the requests before it) * hs_units, each (kv head, sub) in turn.
struct KvCut {
  long long total;  // tiles of all requests, times units per request
  int ctas;         // CTAs with work
};
VDEV long long cut_at(long long total, int ctas, int i) { return total * i / ctas; }
// the CTA whose stretch holds u: the largest i with cut_at(i) <= u
VDEV int cut_owner(long long total, int ctas, long long u) { return (int)(((u + 1) * ctas - 1) / total); }

// a producer's or consumer's place on the line
template <int TILE>
struct KvWalk {
  int seq, unit, tile, len, ntile;  // unit = kv head * nsub + sub
  long long left;                   // tiles left in this CTA's stretch
  VDEV void load(const KvAttnParams& p) {
    len = kv_len_of(p, seq);
    ntile = (len + TILE - 1) / TILE;
  }
  // tiles of the current pair that belong to this CTA
  VDEV int count() const { return (int)min((long long)(ntile - tile), left); }
  VDEV void next(const KvAttnParams& p) {  // past the current pair's tiles
    left -= count();
    tile = 0;
    if (left <= 0 || ++unit < p.G * p.nsub) return;
    unit = 0;
    do {
      seq++;
      load(p);
    } while (ntile == 0);  // left > 0: a request with tiles follows
  }
};

// Finds the CTA's stretch: block-wide, every thread returns the same walk.
template <int TILE>
VDEV KvWalk<TILE> kv_start(const KvAttnParams& p, long long* red, int* found) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5, nt = blockDim.x;
  const int units = p.G * p.nsub;
  const int per = (p.n_seqs + nt - 1) / nt, lo = min(p.n_seqs, tid * per), hi = min(p.n_seqs, lo + per);
  long long sum = 0;
  for (int s = lo; s < hi; s++) sum += (kv_len_of(p, s) + TILE - 1) / TILE;
  long long inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 31) red[warp] = inc;
  __syncthreads();
  long long before = 0, total = 0;
  for (int w = 0; w < nw; w++) {
    if (w < warp) before += red[w];
    total += red[w];
  }
  before += inc - sum;
  total *= units;
  KvWalk<TILE> k;
  const int ctas = (int)min((long long)p.ctas, total);
  k.left = 0;
  k.seq = k.unit = k.tile = k.len = k.ntile = 0;
  if ((int)blockIdx.x >= ctas) return k;
  const long long u0 = cut_at(total, ctas, blockIdx.x), u1 = cut_at(total, ctas, blockIdx.x + 1);
  if (u0 >= before * units && u0 < (before + sum) * units) {  // one thread
    long long b = before * units;
    for (int s = lo; s < hi; s++) {
      const int n = (kv_len_of(p, s) + TILE - 1) / TILE;
      if (u0 < b + (long long)n * units) {
        found[0] = s;
        found[1] = (int)((u0 - b) / n);
        found[2] = (int)((u0 - b) % n);
        break;
      }
      b += (long long)n * units;
    }
  }
  __syncthreads();
  k.seq = found[0];
  k.unit = found[1];
  k.tile = found[2];
  k.left = u1 - u0;
  k.load(p);
  return k;
}

VDEV void tma_load_4d(void* dst, const CUtensorMap* map, int x, int pos, int head, int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          smem_addr(dst)),
      "l"(map), "r"(x), "r"(pos), "r"(head), "r"(page), "r"(smem_addr(bar))
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
VDEV float2 unpack2(uint32_t u, __nv_bfloat16) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u)); }
template <class TC>
VDEV uint32_t pack2_rest(uint32_t hi, float a, float b) {
  const float2 f = unpack2(hi, TC());
  return pack2(a - f.x, b - f.y, TC());
}

// a product and that of the rests; an infinite one stands for itself (its
// rest is an infinity of either sign, or NaN)
VDEV float add_rest(float v, float rest) { return fabsf(v) < INFINITY ? v + rest : v; }

VDEV void consumer_sync() { asm volatile("bar.sync 1, %0;" ::"r"(kPaConsumers) : "memory"); }

// The shared state that kernel and producer agree on.
struct KvRing {
  uint64_t full[kPaStages], empty[kPaStages];
  long long red[kPaThreads / 32];
  int found[3];
  int abort;
};

// ---- producer warp -----------------------------------------------------------
template <class TC, int HS>
VDEV void kv_produce(const KvAttnParams& p, const CUtensorMap* mk, const CUtensorMap* mv,
                     KvWalk<kv_tile<TC>()> w, KvRing* ring, uint8_t* stages) {
  constexpr int TILE = kv_tile<TC>(), NB = HS * (int)sizeof(TC) / 128, XE = 128 / (int)sizeof(TC);
  constexpr int BOX = TILE * 128;  // bytes of one 128-byte column of a tile
  const int lane = threadIdx.x & 31;
  const int page = 1 << p.ps_shift, ppt = max(1, TILE >> p.ps_shift), rows = min(page, TILE);
  int it = 0;
  for (; w.left > 0; w.next(p)) {
    const int g = w.unit / p.nsub, n = w.count();
    const int32_t* row = p.nsel ? p.table + ((int64_t)w.seq * p.G + g) * p.nsel : p.table + (int64_t)w.seq * p.table_stride;
    const int npages = (w.len + page - 1) >> p.ps_shift;
    const auto page_of = [&](int t) { return (t * TILE >> p.ps_shift) + (lane < ppt ? lane : 0); };
    int pi = page_of(w.tile);
    int id = pi < npages ? row[pi] : 0;  // one tile ahead of its use
    for (int t = w.tile; t < w.tile + n; t++, it++) {
      const int mine = id, mpi = pi;
      if (t + 1 < w.tile + n) {
        pi = page_of(t + 1);
        id = pi < npages ? row[pi] : 0;
      }
      const bool has = lane < ppt && mpi < npages;
      const int cnt = __popc(__ballot_sync(0xffffffffu, has));
      const int slot = it % kPaStages;
      int ok = 1;
      if (it >= kPaStages) ok = mbar_wait_warp(&ring->empty[slot], ((uint32_t)(it / kPaStages) & 1u) ^ 1u, &ring->abort);
      if (!ok) goto drain;
      if (lane == 0) mbar_arrive_expect_tx(&ring->full[slot], (uint32_t)(cnt * rows * HS * (int)sizeof(TC) * 2));
      __syncwarp();
      if (has) {
        int pg = mine;
        if (pg < 0 || pg >= p.n_pages) {
          set_error(p.err, VIREO_ERR_ARG);
          pg = p.n_pages;  // outside the map: zeros
        }
        const int off = (t * TILE) & (page - 1);  // 0 when a tile holds whole pages
        uint8_t* dk = stages + (size_t)slot * kv_stage_bytes<TC, HS>() + lane * rows * 128;
        uint8_t* dv = dk + NB * BOX;
#pragma unroll
        for (int b = 0; b < NB; b++) tma_load_4d(dk + b * BOX, mk, b * XE, off, g, pg, &ring->full[slot]);
#pragma unroll
        for (int b = 0; b < NB; b++) tma_load_4d(dv + b * BOX, mv, b * XE, off, g, pg, &ring->full[slot]);
      }
    }
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

// ---- 16-bit cache: tensor cores ------------------------------------------------
template <class TA, class TC, int HS>
VDEV void kv_consume_mma(const KvAttnParams& p, KvWalk<64> w, KvRing* ring, uint8_t* stages, float* merge) {
  constexpr int TILE = 64, KS = HS / 16, NT = HS / 8;
  constexpr bool QSPLIT = sizeof(TA) == 4;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
  int it = 0;
  for (bool first = true; w.left > 0; w.next(p), first = false) {
    const int kh = w.unit / p.nsub, sub = w.unit - kh * p.nsub, n = w.count();
    const int nh = min(kPaHeads, p.R - sub * kPaHeads);
    const int h = kh * p.R + sub * kPaHeads + g;  // this lane's q head, if g < nh
    // q as A fragments: row g the value in the cache's type, row g + 8 what
    // that left of an fp32 value.  An fp32 row is first scaled by the power
    // of two that brings its largest value to [1, 2), so that neither half
    // leaves the type's range; the scores take it back.
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
        // exponent of mx, within what a power of two and its inverse can hold
        const int e = mx > 0.f && mx < INFINITY ? min(max(ilogbf(mx), -100), 100) : 0;
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
    float o[NT][4];
#pragma unroll
    for (int j = 0; j < NT; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    float m_run = -INFINITY, l_run = 0.f;
    const int wr = 16 * warp;  // this warp's rows of a tile
#pragma unroll 1
    for (int t = w.tile; t < w.tile + n; t++, it++) {
      const int slot = it % kPaStages;
      const bool ok = mbar_wait_warp(&ring->full[slot], (uint32_t)(it / kPaStages) & 1u, &ring->abort);
      if (!ok && lane == 0) {
        ring->abort = 1;
        set_error(p.err, VIREO_ERR_TIMEOUT);
      }
      uint8_t* st = stages + (size_t)slot * kv_stage_bytes<TC, HS>();
      const int rows = min(TILE, w.len - t * TILE);
      if (ok && wr < rows) {
        uint8_t* kt = st;
        uint8_t* vt = st + TILE * HS * 2;
        if (wr + 16 > rows) {
          // value rows behind the last position: zeros, since their weight of
          // zero does not cancel a NaN
          for (int r = rows; r < wr + 16; r++)
            for (int c = lane; c < HS / 8; c += 32)
              *reinterpret_cast<uint4*>(vt + kv_at<TILE>(r, c)) = make_uint4(0u, 0u, 0u, 0u);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the stage is filled by copies again
          __syncwarp();
        }
        float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < KS; s += 2) {
          uint32_t b[2][4];
#pragma unroll
          for (int j = 0; j < 2; j++)
            ldsm_x4(kt + kv_at<TILE>(wr + 8 * j + (lane & 7), 2 * s + (lane >> 3)), b[j][0], b[j][1], b[j][2], b[j][3]);
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
          mma_kv(s0, a1, b[0][2], b[0][3], TC());
          mma_kv(s1, a1, b[1][2], b[1][3], TC());
        }
        if constexpr (QSPLIT) {
          s0[0] = add_rest(s0[0], s0[2]);
          s0[1] = add_rest(s0[1], s0[3]);
          s1[0] = add_rest(s1[0], s1[2]);
          s1[1] = add_rest(s1[1], s1[3]);
        }
        // this lane's positions: wr + 2 t4 (+1) and wr + 8 + 2 t4 (+1)
        const int q0 = wr + 2 * t4;
        const float v0 = q0 < rows ? s0[0] * qs : -INFINITY, v1 = q0 + 1 < rows ? s0[1] * qs : -INFINITY;
        const float v2 = q0 + 8 < rows ? s1[0] * qs : -INFINITY, v3 = q0 + 9 < rows ? s1[1] * qs : -INFINITY;
        float mt = fmaxf(fmaxf(v0, v1), fmaxf(v2, v3));
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
        const float m_new = fmaxf(m_run, mt);
        // scores of -inf alone leave the maximum at -inf: subtract 0 then
        const float m_sub = m_new == -INFINITY ? 0.f : m_new;
        if (__any_sync(0xffffffffu, m_new > m_run)) {
          const float alpha = exp2f(m_run - m_sub);
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
        const float e0 = exp2f(v0 - m_sub), e1 = exp2f(v1 - m_sub), e2 = exp2f(v2 - m_sub), e3 = exp2f(v3 - m_sub);
        l_run += (e0 + e1) + (e2 + e3);
        uint32_t pa[4];
        pa[0] = pack2(e0, e1, TC());
        pa[1] = pack2_rest<TC>(pa[0], e0, e1);
        pa[2] = pack2(e2, e3, TC());
        pa[3] = pack2_rest<TC>(pa[2], e2, e3);
#pragma unroll
        for (int j = 0; j < NT; j += 2) {
          uint32_t b0, b1, b2, b3;
          ldsm_x4_trans(vt + kv_at<TILE>(wr + (lane & 7) + 8 * ((lane >> 3) & 1), j + (lane >> 4)), b0, b1, b2, b3);
          mma_kv(o[j], pa, b0, b1, TC());
          mma_kv(o[j + 1], pa, b2, b3, TC());
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&ring->empty[slot]);
    }
    // ---- the warps' states joined, in pairs, through shared memory ------------
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);
#pragma unroll
    for (int j = 0; j < NT; j++) {
      o[j][0] = add_rest(o[j][0], o[j][2]);
      o[j][1] = add_rest(o[j][1], o[j][3]);
    }
    // each lane's registers to the same lane of the warp that takes them in
    const auto put = [&](float* b) {
#pragma unroll
      for (int j = 0; j < NT; j++)
        *reinterpret_cast<float2*>(b + 2 * (j * 32 + lane)) = make_float2(o[j][0], o[j][1]);
      b[2 * NT * 32 + lane] = m_run;
      b[2 * NT * 32 + 32 + lane] = l_run;
    };
    const auto take = [&](const float* b) {
      const float m2 = b[2 * NT * 32 + lane], l2 = b[2 * NT * 32 + 32 + lane];
      const float m_new = fmaxf(m_run, m2), m_sub = m_new == -INFINITY ? 0.f : m_new;
      const float f1 = exp2f(m_run - m_sub), f2 = exp2f(m2 - m_sub);
#pragma unroll
      for (int j = 0; j < NT; j++) {
        const float2 v = *reinterpret_cast<const float2*>(b + 2 * (j * 32 + lane));
        o[j][0] = o[j][0] * f1 + v.x * f2;
        o[j][1] = o[j][1] * f1 + v.y * f2;
      }
      l_run = l_run * f1 + l2 * f2;
      m_run = m_new;
    };
    constexpr int MB = 2 * NT * 32 + 64;
    if (warp >= 2) put(merge + (warp - 2) * MB);
    consumer_sync();
    if (warp < 2) take(merge + warp * MB);
    consumer_sync();
    if (warp == 1) put(merge);
    consumer_sync();
    if (warp == 0) {
      take(merge);
      const bool whole = w.tile == 0 && n == w.ntile;
      if (g < nh) {
        if (whole) {
          const float r = l_run > 0.f ? 1.0f / l_run : (l_run == 0.f ? 0.f : l_run);  // a NaN stays one
          TA* out = reinterpret_cast<TA*>(p.out) + (int64_t)w.seq * p.out_stride + (int64_t)h * HS + 2 * t4;
#pragma unroll
          for (int j = 0; j < NT; j++) {
            const float v[2] = {o[j][0] * r, o[j][1] * r};
            store_f<2>(out + 8 * j, v);
          }
        } else {
          float* b = p.part + ((size_t)(2 * blockIdx.x + (first ? 0 : 1)) * kPaHeads + g) * (HS + 2);
#pragma unroll
          for (int j = 0; j < NT; j++)
            *reinterpret_cast<float2*>(b + 8 * j + 2 * t4) = make_float2(o[j][0], o[j][1]);
          if (t4 == 0) {
            b[HS] = m_run;
            b[HS + 1] = l_run;
          }
        }
      }
    }
    consumer_sync();  // merge is free again
  }
}

// ---- fp32 cache: CUDA cores ----------------------------------------------------
// A warp takes eight of a tile's positions.  Scores: lane (position lane & 7,
// quarter lane >> 3) multiplies every fourth 16-byte chunk of its key with
// the RT q heads in shared memory; the quarters are added by shuffles.
// Values: lane i owns 16-byte chunk i (mod chunks of a row) of the output and
// adds weight x value over the positions.
template <int HS, int RT>
VDEV void kv_consume_f32(const KvAttnParams& p, KvWalk<32> w, KvRing* ring, uint8_t* stages, float* merge) {
  constexpr int TILE = 32, CH = HS / 4;  // chunks of a row
  constexpr int PS = CH < 32 ? 32 / CH : 1, NC = CH < 32 ? 1 : CH / 32;  // positions side by side, chunks per lane
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pp = lane & 7, qd = lane >> 3;
  float* sq = merge;                                   // [RT][HS]
  float* sp = sq + RT * HS + warp * (8 * RT + RT);     // per warp: [8][RT] weights, [RT] rescales
  float* mb = sq + RT * HS + kPaWarps * (8 * RT + RT); // [2][RT * NC * 4 + 2 * RT][32]
  constexpr int MB = (RT * NC * 4 + 2 * RT) * 32;
  int it = 0;
  for (bool first = true; w.left > 0; w.next(p), first = false) {
    const int kh = w.unit / p.nsub, sub = w.unit - kh * p.nsub, n = w.count();
    const int nh = min(RT, p.R - sub * kPaHeads), h0 = kh * p.R + sub * kPaHeads;
    const float* q = reinterpret_cast<const float*>(p.q) + (int64_t)w.seq * p.q_stride + (int64_t)h0 * HS;
    for (int i = threadIdx.x * 4; i < RT * HS; i += kPaConsumers * 4)
      *reinterpret_cast<float4*>(sq + i) =
          i < nh * HS ? *reinterpret_cast<const float4*>(q + i) : make_float4(0.f, 0.f, 0.f, 0.f);
    consumer_sync();
    float o[RT][NC * 4], m_run[RT], l_run[RT];
#pragma unroll
    for (int r = 0; r < RT; r++) {
      m_run[r] = -INFINITY;
      l_run[r] = 0.f;
#pragma unroll
      for (int j = 0; j < NC * 4; j++) o[r][j] = 0.f;
    }
    const int wr = 8 * warp;
#pragma unroll 1
    for (int t = w.tile; t < w.tile + n; t++, it++) {
      const int slot = it % kPaStages;
      const bool ok = mbar_wait_warp(&ring->full[slot], (uint32_t)(it / kPaStages) & 1u, &ring->abort);
      if (!ok && lane == 0) {
        ring->abort = 1;
        set_error(p.err, VIREO_ERR_TIMEOUT);
      }
      const uint8_t* kt = stages + (size_t)slot * kv_stage_bytes<float, HS>();
      const uint8_t* vt = kt + TILE * HS * 4;
      const int rows = min(TILE, w.len - t * TILE);
      if (ok && wr < rows) {
        float s[RT];
#pragma unroll
        for (int r = 0; r < RT; r++) s[r] = 0.f;
#pragma unroll
        for (int i = 0; i < CH / 4; i++) {
          const int c = 4 * i + qd;
          const float4 k = *reinterpret_cast<const float4*>(kt + kv_at<TILE>(wr + pp, c));
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
            const float a = exp2f(m_old[r] - (m_run[r] == -INFINITY ? 0.f : m_run[r]));
            l_run[r] *= a;
#pragma unroll
            for (int j = 0; j < NC * 4; j++) o[r][j] *= a;
          }
        }
#pragma unroll
        for (int r = 0; r < RT; r++) {
          const float e = exp2f(s[r] - (m_run[r] == -INFINITY ? 0.f : m_run[r]));
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
              const float4 v = *reinterpret_cast<const float4*>(vt + kv_at<TILE>(wr + pos, (lane % (CH < 32 ? CH : 32)) + 32 * c));
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
      if (lane == 0) mbar_arrive(&ring->empty[slot]);
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
    const auto put = [&](float* b) {
#pragma unroll
      for (int r = 0; r < RT; r++) {
#pragma unroll
        for (int j = 0; j < NC * 4; j++) b[(r * (NC * 4 + 2) + j) * 32 + lane] = o[r][j];
        b[(r * (NC * 4 + 2) + NC * 4) * 32 + lane] = m_run[r];
        b[(r * (NC * 4 + 2) + NC * 4 + 1) * 32 + lane] = l_run[r];
      }
    };
    const auto take = [&](const float* b) {
#pragma unroll
      for (int r = 0; r < RT; r++) {
        const float m2 = b[(r * (NC * 4 + 2) + NC * 4) * 32 + lane], l2 = b[(r * (NC * 4 + 2) + NC * 4 + 1) * 32 + lane];
        const float m_new = fmaxf(m_run[r], m2), m_sub = m_new == -INFINITY ? 0.f : m_new;
        const float f1 = exp2f(m_run[r] - m_sub), f2 = exp2f(m2 - m_sub);
#pragma unroll
        for (int j = 0; j < NC * 4; j++) o[r][j] = o[r][j] * f1 + b[(r * (NC * 4 + 2) + j) * 32 + lane] * f2;
        l_run[r] = l_run[r] * f1 + l2 * f2;
        m_run[r] = m_new;
      }
    };
    if (warp >= 2) put(mb + (warp - 2) * MB);
    consumer_sync();
    if (warp < 2) take(mb + warp * MB);
    consumer_sync();
    if (warp == 1) put(mb);
    consumer_sync();
    if (warp == 0) {
      take(mb);
      const bool whole = w.tile == 0 && n == w.ntile;
      const int col = (lane % (CH < 32 ? CH : 32)) * 4;
      if (CH >= 32 || lane < CH)
#pragma unroll
        for (int r = 0; r < RT; r++) {
          if (r >= nh) break;
          if (whole) {
            const float f = l_run[r] > 0.f ? 1.0f / l_run[r] : (l_run[r] == 0.f ? 0.f : l_run[r]);
            float* out = reinterpret_cast<float*>(p.out) + (int64_t)w.seq * p.out_stride + (int64_t)(h0 + r) * HS + col;
#pragma unroll
            for (int c = 0; c < NC; c++)
              *reinterpret_cast<float4*>(out + 128 * c) =
                  make_float4(o[r][4 * c] * f, o[r][4 * c + 1] * f, o[r][4 * c + 2] * f, o[r][4 * c + 3] * f);
          } else {
            float* b = p.part + ((size_t)(2 * blockIdx.x + (first ? 0 : 1)) * kPaHeads + r) * (HS + 2);
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
              for (int j = 0; j < 4; j++) b[128 * c + col + j] = o[r][4 * c + j];
            if (lane == 0) {
              b[HS] = m_run[r];
              b[HS + 1] = l_run[r];
            }
          }
        }
    }
    consumer_sync();  // merge and sq are free again
  }
}

template <class TC, int HS, int RT>
__host__ __device__ constexpr int kv_merge_floats() {
  if (sizeof(TC) == 2) return 2 * (2 * (HS / 8) * 32 + 64);
  constexpr int NC = HS / 4 < 32 ? 1 : HS / 128;
  return RT * HS + kPaWarps * 9 * RT + 2 * (RT * NC * 4 + 2 * RT) * 32;
}
template <class TC, int HS, int RT>
constexpr int kv_attn_smem() {
  return 1024 + kPaStages * kv_stage_bytes<TC, HS>() + kv_merge_floats<TC, HS, RT>() * 4;
}

template <class TA, class TC, int HS, int RT>
__global__ void __launch_bounds__(kPaThreads, HS == 256 ? 1 : 2)
    kv_attn_kernel(const __grid_constant__ KvAttnParams p, const __grid_constant__ CUtensorMap mk,
                   const __grid_constant__ CUtensorMap mv) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ KvRing ring;
  uint8_t* stages = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);  // swizzle atoms of 1024 bytes
  float* merge = reinterpret_cast<float*>(stages + kPaStages * kv_stage_bytes<TC, HS>());
  if (threadIdx.x == 0) {
    for (int s = 0; s < kPaStages; s++) {
      mbar_init(&ring.full[s], 1);
      mbar_init(&ring.empty[s], kPaWarps);
    }
    ring.abort = 0;
    mbar_fence_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();  // after the wait: the merge may read kv_len before its own
  asm volatile("fence.proxy.async;" ::: "memory");  // pool rows written by the kernels before this one
  const auto w = kv_start<kv_tile<TC>()>(p, ring.red, ring.found);
  if (w.left <= 0) return;
  if (threadIdx.x >= kPaConsumers) {
    kv_produce<TC, HS>(p, &mk, &mv, w, &ring, stages);
  } else if constexpr (sizeof(TC) == 2) {
    kv_consume_mma<TA, TC, HS>(p, w, &ring, stages, merge);
  } else {
    kv_consume_f32<HS, RT>(p, w, &ring, stages, merge);
  }
}

// Joins the partial states of a (request, q head) that several CTAs share:
// M = max m_c, out = sum 2^(m_c - M) acc_c / sum 2^(m_c - M) l_c, in CTA
// order.  Also writes the zeros of requests without positions.
constexpr int kMergeThreads = 128;
template <class TA, int TILE>
__global__ void __launch_bounds__(kMergeThreads) kv_merge_kernel(const __grid_constant__ KvAttnParams p, int hs) {
  __shared__ long long red[2][kMergeThreads / 32];
  extern __shared__ float wgt[];  // [ctas] weights of the partial states
  __shared__ float fred[2][kMergeThreads / 32];
  const int seq = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int units = p.G * p.nsub;
  // where the request's tiles start on the line, and the line's length
  long long before = 0, all = 0;
  for (int s = tid; s < p.n_seqs; s += kMergeThreads) {
    const int n = (kv_len_of(p, s) + TILE - 1) / TILE;
    all += n;
    if (s < seq) before += n;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    all += __shfl_xor_sync(0xffffffffu, all, o);
  }
  if (lane == 0) {
    red[0][warp] = before;
    red[1][warp] = all;
  }
  __syncthreads();
  before = all = 0;
#pragma unroll
  for (int i = 0; i < kMergeThreads / 32; i++) {
    before += red[0][i];
    all += red[1][i];
  }
  const int len = kv_len_of(p, seq);
  TA* out = reinterpret_cast<TA*>(p.out) + (int64_t)seq * p.out_stride + (int64_t)h * hs;
  pdl_wait();
  if (len == 0) {
    for (int i = tid * 4; i < hs; i += kMergeThreads * 4) {
      const float z[4] = {0.f, 0.f, 0.f, 0.f};
      store_f<4>(out + i, z);
    }
    return;
  }
  const long long total = all * units;
  const int ctas = (int)min((long long)p.ctas, total);
  const int kh = h / p.R, r = h - kh * p.R, unit = kh * p.nsub + r / kPaHeads, g = r % kPaHeads;
  const long long n = (len + TILE - 1) / TILE, u0 = before * units + unit * n;
  const int c0 = cut_owner(total, ctas, u0), c1 = cut_owner(total, ctas, u0 + n - 1), nc = c1 - c0 + 1;
  if (nc == 1) return;  // finished by its CTA
  // the pair is the first of every CTA but, perhaps, of c0
  const int slot0 = cut_at(total, ctas, c0) == u0 ? 0 : 1;
  const auto state = [&](int i) {
    return p.part + ((size_t)(2 * (c0 + i) + (i ? 0 : slot0)) * kPaHeads + g) * (hs + 2);
  };
  float M = -INFINITY;
  for (int i = tid; i < nc; i += kMergeThreads) M = fmaxf(M, __ldcg(state(i) + hs));
#pragma unroll
  for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if (lane == 0) fred[0][warp] = M;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kMergeThreads / 32; i++) M = fmaxf(M, fred[0][i]);
  const float m_sub = M == -INFINITY ? 0.f : M;
  float L = 0.f;
  for (int i = tid; i < nc; i += kMergeThreads) {
    const float f = exp2f(__ldcg(state(i) + hs) - m_sub);
    wgt[i] = f;
    L += f * __ldcg(state(i) + hs + 1);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
  if (lane == 0) fred[1][warp] = L;
  __syncthreads();
  L = 0.f;
#pragma unroll
  for (int i = 0; i < kMergeThreads / 32; i++) L += fred[1][i];
  const float f = L > 0.f ? 1.0f / L : (L == 0.f ? 0.f : L);
  for (int e = tid; e < hs; e += kMergeThreads) {
    float acc = 0.f;
    int i = 0;
    for (; i + 8 <= nc; i += 8) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = __ldcg(state(i + j) + e);
#pragma unroll
      for (int j = 0; j < 8; j++) acc += v[j] * wgt[i + j];
    }
    for (; i < nc; i++) acc += __ldcg(state(i) + e) * wgt[i];
    out[e] = from_f<TA>(acc * f);
  }
}

// ---------------------------------------------------------------------------
// Block selection.
//
// kv_score_kernel: a lane group of LPR lanes holds a page's mean key, E
// values each, and the kv head's q values for the same dimensions in
// registers as doubles (up to eight heads at a time); products of a 16-bit or
// fp32 key with an fp32 query are exact in 64 bits and the sum's error is
// 2^-53 relative, so the order of the additions does not decide between
// pages.  The per-head sums are reduced over the group by halving (heads x
// lanes), then the maximum over heads becomes a sortable 64-bit key.
// kv_select_kernel: one CTA per (request, kv head) finds the n_top-th
// largest key by radix selection, 11 bits at a time, stopping as soon as the
// keys above and at the current prefix are exactly as many as wanted, and
// writes the chosen pages in rising order, as indices and as pool pages.
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
template <class TA, class TC, int HS>
__global__ void __launch_bounds__(kScoreThreads) kv_score_kernel(const __grid_constant__ KvSelectParams p, int per) {
  constexpr int E = 8, LPR = HS / E, GPB = kScoreThreads / LPR;
  pdl_wait();
  pdl_launch_dependents();
  const int seq = blockIdx.z, g = blockIdx.y;
  const int np = select_pages(p, seq);
  if (np <= p.nsel) return;
  const int lo = p.n_sink + blockIdx.x * per, hi = min(np - p.n_window, lo + per);
  if (lo >= hi) return;
  const int grp = threadIdx.x / LPR, l = threadIdx.x % LPR;
  const unsigned mask = LPR == 32 ? 0xffffffffu : ((1u << LPR) - 1u) << ((threadIdx.x & 31) / LPR * LPR);
  const int32_t* row = p.table + (int64_t)seq * p.table_stride;
  uint64_t* keys = p.keys + ((int64_t)seq * p.G + g) * p.max_pages;
  for (int r0 = 0; r0 < p.R; r0 += 8) {
    double q[8][E];
#pragma unroll
    for (int r = 0; r < 8; r++) {
      float v[E];
#pragma unroll
      for (int e = 0; e < E; e++) v[e] = 0.f;
      if (r0 + r < p.R)
        load_f<E>((const TA*)p.q + (int64_t)seq * p.q_stride + (int64_t)(g * p.R + r0 + r) * HS + l * E, v);
#pragma unroll
      for (int e = 0; e < E; e++) q[r][e] = (double)v[e];
    }
    for (int pg = lo + grp; pg < hi; pg += GPB) {
      const int id = row[pg];
      float k[E];
      if (id >= 0 && id < p.n_pages) {
        load_f<E>((const TC*)p.means + ((int64_t)id * p.G + g) * HS + l * E, k);
      } else {
        set_error(p.err, VIREO_ERR_ARG);
#pragma unroll
        for (int e = 0; e < E; e++) k[e] = 0.f;
      }
      double s[8];
#pragma unroll
      for (int r = 0; r < 8; r++) s[r] = 0.0;
#pragma unroll
      for (int e = 0; e < E; e++) {
        const double kd = (double)k[e];
#pragma unroll
        for (int r = 0; r < 8; r++) s[r] = fma(q[r][e], kd, s[r]);
      }
      // LPR lanes x 8 heads -> each lane one head's sum (LPR >= 8): lanes
      // whose bit is set keep the upper half of the heads
#pragma unroll
      for (int b = 4; b >= 1; b >>= 1) {
        const bool upper = (l & b) != 0;
#pragma unroll
        for (int r = 0; r < b; r++) {
          const double send = upper ? s[r] : s[r + b], keep = upper ? s[r + b] : s[r];
          s[r] = keep + __shfl_xor_sync(mask, send, b);
        }
      }
#pragma unroll
      for (int o = 8; o < LPR; o <<= 1) s[0] += __shfl_xor_sync(mask, s[0], o);
      // lane l now has head r0 + (l & 7)
      uint64_t key = r0 + (l & 7) < p.R ? sort_key(s[0]) : 0ull;
#pragma unroll
      for (int o = 4; o >= 1; o >>= 1) {
        const uint64_t other = __shfl_xor_sync(mask, key, o);
        key = other > key ? other : key;
      }
      if (l == 0) keys[pg] = r0 ? max(key, keys[pg]) : key;
    }
  }
}

constexpr int kSelThreads = 512;
constexpr int kSelBits = 11, kSelBins = 1 << kSelBits;
constexpr int kSelCache = 4096;  // keys held in shared memory

__global__ void __launch_bounds__(kSelThreads) kv_select_kernel(const __grid_constant__ KvSelectParams p) {
  __shared__ unsigned int hist[kSelBins];
  __shared__ uint64_t cache[kSelCache];
  __shared__ int wsum[2][kSelThreads / 32];
  __shared__ int pick[2];
  pdl_wait();
  pdl_launch_dependents();
  const int seq = blockIdx.y, g = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
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
  for (int i = tid; i < p.n_sink; i += kSelThreads) put(i, i);
  for (int i = tid; i < p.n_window; i += kSelThreads) put(p.n_sink + p.n_top + i, np - p.n_window + i);
  if (p.n_top == 0) return;
  const int m = np - p.n_sink - p.n_window;  // candidates, more than n_top
  const uint64_t* keys = p.keys + ((int64_t)seq * p.G + g) * p.max_pages + p.n_sink;
  for (int i = tid; i < min(m, kSelCache); i += kSelThreads) cache[i] = __ldcg(keys + i);
  const auto key = [&](int i) { return i < kSelCache ? cache[i] : __ldcg(keys + i); };
  // radix selection: keys with the bits of `prefix` above `shift` are still
  // in question; `want` of them are to be taken
  uint64_t prefix = 0;
  int want = p.n_top, shift = 64, equal = m;
  while (shift > 0 && equal > want) {
    const int bits = min(kSelBits, shift), next = shift - bits;
    for (int i = tid; i < kSelBins; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < m; i += kSelThreads) {
      const uint64_t k = key(i);
      if (shift == 64 || (k >> shift) == (prefix >> shift))
        atomicAdd(&hist[(int)(k >> next) & ((1 << bits) - 1)], 1u);
    }
    __syncthreads();
    // thread i owns the bins [BPT * i, BPT * (i + 1)) counted from the top
    constexpr int BPT = kSelBins / kSelThreads;
    int c[BPT], sum = 0;
#pragma unroll
    for (int j = 0; j < BPT; j++) {
      const int bin = (1 << bits) - 1 - (tid * BPT + j);
      c[j] = bin >= 0 ? (int)hist[bin] : 0;
      sum += c[j];
    }
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    if (lane == 31) wsum[0][warp] = inc;
    __syncthreads();
    for (int w = 0; w < warp; w++) inc += wsum[0][w];
    int above = inc - sum;  // keys in higher bins
    if (above < want && inc >= want) {
#pragma unroll
      for (int j = 0; j < BPT; j++) {
        if (above < want && above + c[j] >= want) {
          pick[0] = (1 << bits) - 1 - (tid * BPT + j);
          pick[1] = above;
          wsum[1][0] = c[j];
          break;
        }
        above += c[j];
      }
    }
    __syncthreads();
    prefix |= (uint64_t)pick[0] << next;
    want -= pick[1];
    equal = wsum[1][0];
    shift = next;
    __syncthreads();
  }
  // taken: keys above the prefix, and the first `want` at it (all of them,
  // or the lowest pages of equal keys)
  __syncthreads();
  int base_hi = 0, base_eq = 0;
  for (int b = 0; b < m; b += kSelThreads) {
    const int i = b + tid;
    bool hi = false, eq = false;
    if (i < m) {
      const uint64_t k = key(i);
      const uint64_t top = shift < 64 ? k >> shift : 0, ptop = shift < 64 ? prefix >> shift : 0;
      hi = top > ptop;
      eq = top == ptop;
    }
    const unsigned bh = __ballot_sync(0xffffffffu, hi), be = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) {
      wsum[0][warp] = __popc(bh);
      wsum[1][warp] = __popc(be);
    }
    __syncthreads();
    int nh = base_hi, ne = base_eq;
    for (int w = 0; w < kSelThreads / 32; w++) {
      if (w < warp) {
        nh += wsum[0][w];
        ne += wsum[1][w];
      }
      base_hi += wsum[0][w];
      base_eq += wsum[1][w];
    }
    nh += __popc(bh & ((1u << lane) - 1u));
    ne += __popc(be & ((1u << lane) - 1u));
    if (hi || (eq && ne < want)) put(p.n_sink + nh + min(ne, want), p.n_sink + i);
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static int kv_make_map(const gguf_kv_desc& d, CUtensorMap* m, void* base) {
  void* f = nullptr;
  cudaDriverEntryPointQueryResult q;
  if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
      q != cudaDriverEntryPointSuccess) {
    cudaGetLastError();
    return VIREO_ERR_UNSUPPORTED;
  }
  const int el = kv_type_size(d.kv_type), tile = el == 4 ? 32 : 64;
  const cuuint64_t dims[4] = {(cuuint64_t)d.head_size, (cuuint64_t)d.page_size, (cuuint64_t)d.n_kv_heads,
                              (cuuint64_t)d.n_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)d.pos_stride * el, (cuuint64_t)d.head_stride * el,
                                 (cuuint64_t)d.page_stride * el};
  const cuuint32_t box[4] = {(cuuint32_t)(128 / el), (cuuint32_t)std::min(d.page_size, tile), 1, 1};
  const cuuint32_t es[4] = {1, 1, 1, 1};
  const CUtensorMapDataType ty = d.kv_type == KV_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                 : d.kv_type == KV_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                       : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUresult r = ((EncodeTiledFn)f)(m, ty, 4, base, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? VIREO_OK : VIREO_ERR_UNSUPPORTED;
}

struct KvKernel {
  const void* fn;
  int smem;
};
template <class TA, class TC, int HS, int RT>
static KvKernel kv_kernel() {
  return {reinterpret_cast<const void*>(&kv_attn_kernel<TA, TC, HS, RT>), kv_attn_smem<TC, HS, RT>()};
}
template <class TA, class TC>
static KvKernel kv_kernel_h(int hs) {
  switch (hs) {
    case 64: return kv_kernel<TA, TC, 64, kPaHeads>();
    case 128: return kv_kernel<TA, TC, 128, kPaHeads>();
    default: return kv_kernel<TA, TC, 256, kPaHeads>();
  }
}
// fp32 cache: the smallest of 1, 2, 4, 8 heads that holds the group
template <int HS>
static KvKernel kv_kernel_f32(int R) {
  if (R == 1) return kv_kernel<float, float, HS, 1>();
  if (R == 2) return kv_kernel<float, float, HS, 2>();
  if (R <= 4) return kv_kernel<float, float, HS, 4>();
  return kv_kernel<float, float, HS, 8>();
}
static KvKernel kv_kernel_for(const gguf_kv_desc& d) {
  const int R = d.n_heads / d.n_kv_heads;
  if (d.act_type == KV_BF16) return kv_kernel_h<__nv_bfloat16, __nv_bfloat16>(d.head_size);
  if (d.act_type == KV_F16) return kv_kernel_h<__half, __half>(d.head_size);
  if (d.kv_type == KV_F16) return kv_kernel_h<float, __half>(d.head_size);
  return d.head_size == 64 ? kv_kernel_f32<64>(R) : d.head_size == 128 ? kv_kernel_f32<128>(R) : kv_kernel_f32<256>(R);
}

// CTAs of the attention kernel that the workspace has room for: two to an SM
// of up to 256 SMs; the launch takes as many as are resident
constexpr int kPaMaxCtas = 512;

template <class TA, class TC>
static const void* score_kernel_h(int hs) {
  switch (hs) {
    case 64: return reinterpret_cast<const void*>(&kv_score_kernel<TA, TC, 64>);
    case 128: return reinterpret_cast<const void*>(&kv_score_kernel<TA, TC, 128>);
    default: return reinterpret_cast<const void*>(&kv_score_kernel<TA, TC, 256>);
  }
}
static const void* score_kernel_for(const gguf_kv_desc& d) {
  if (d.act_type == KV_BF16) return score_kernel_h<__nv_bfloat16, __nv_bfloat16>(d.head_size);
  if (d.act_type == KV_F16) return score_kernel_h<__half, __half>(d.head_size);
  if (d.kv_type == KV_F16) return score_kernel_h<float, __half>(d.head_size);
  return score_kernel_h<float, float>(d.head_size);
}

static int launch_pdl_c(const void* fn, dim3 grid, dim3 block, size_t smem, cudaStream_t s, void** args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelExC(&cfg, fn, args));
}

static size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }
// the workspace: partial states, then with block selection scores and pages
struct KvWs {
  size_t part, keys, phys, total;
};
static KvWs kv_ws(const gguf_kv_desc& d, int n_seqs, int max_pages, int nsel) {
  KvWs w;
  w.part = 0;
  w.keys = up256((size_t)kPaMaxCtas * 2 * kPaHeads * (d.head_size + 2) * 4);
  w.phys = w.keys + (nsel ? up256((size_t)n_seqs * d.n_kv_heads * max_pages * 8) : 0);
  w.total = w.phys + (nsel ? up256((size_t)n_seqs * d.n_kv_heads * nsel * 4) : 0);
  return w;
}

static int kv_attn_check(const gguf_kv* kv, const gguf_kv_attn_args* a) {
  if (!kv || !a || a->n_seqs < 0 || a->max_pages < 1) return VIREO_ERR_ARG;
  const gguf_kv_desc& d = kv->d;
  if ((int64_t)a->max_pages * d.page_size > INT32_MAX) return VIREO_ERR_ARG;
  if (a->n_seqs == 0) return VIREO_OK;
  const int el = kv_type_size(d.act_type);
  const int64_t w = (int64_t)d.n_heads * d.head_size;
  if (!a->q || !a->out || !a->table || !a->kv_len || !a->ws || !kv_aligned(a->q, 16) || !kv_aligned(a->out, 16) ||
      !kv_aligned(a->ws, 256) || !kv_stride_ok(a->q_stride, w, el) || !kv_stride_ok(a->out_stride, w, el) ||
      a->table_stride < a->max_pages || !(a->scale == a->scale))
    return VIREO_ERR_ARG;
  return VIREO_OK;
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
      if ((st = kv_make_map(d, &kv->map_k, d.k)) || (st = kv_make_map(d, &kv->map_v, d.v)) ||
          (st = cuda_status(cudaFuncSetAttribute(k.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, k.smem))) ||
          (st = cuda_status(cudaFuncSetAttribute(k.fn, cudaFuncAttributePreferredSharedMemoryCarveout,
                                                 cudaSharedmemCarveoutMaxShared))) ||
          (st = cuda_status(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&kv->per_sm, k.fn, kPaThreads, k.smem))))
        return st;
      if (kv->per_sm < 1) return VIREO_ERR_UNSUPPORTED;
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
  p.nsub = (p.R + kPaHeads - 1) / kPaHeads;
  p.ps_shift = kv->ps_shift;
  p.nsel = nsel;
  p.scale = (a.scale == 0.f ? 1.0f / sqrtf((float)d.head_size) : a.scale) * kLog2e;
  p.part = (float*)a.ws;
  p.err = c->d_err;
  // no more CTAs than tiles there can be
  const int tile = kv_type_size(d.kv_type) == 4 ? 32 : 64;
  const int64_t most = (int64_t)a.n_seqs * p.G * p.nsub *
                       (((int64_t)(nsel ? std::min(nsel, a.max_pages) : a.max_pages) * d.page_size + tile - 1) / tile);
  p.ctas = (int)std::min<int64_t>(std::min(kPaMaxCtas, c->num_sms * per_sm), most);
  void* args[] = {&p, &mk, &mv};
  if ((st = launch_pdl_c(k.fn, dim3(p.ctas), dim3(kPaThreads), k.smem, s, args))) return st;
  const dim3 grid(a.n_seqs, d.n_heads);
  const size_t msm = (size_t)p.ctas * 4;
  if (d.act_type == KV_BF16)
    return pdl_launch(kv_merge_kernel<__nv_bfloat16, 64>, grid, dim3(kMergeThreads), msm, s, p, d.head_size);
  if (d.act_type == KV_F16)
    return pdl_launch(kv_merge_kernel<__half, 64>, grid, dim3(kMergeThreads), msm, s, p, d.head_size);
  if (d.kv_type == KV_F16)
    return pdl_launch(kv_merge_kernel<float, 64>, grid, dim3(kMergeThreads), msm, s, p, d.head_size);
  return pdl_launch(kv_merge_kernel<float, 32>, grid, dim3(kMergeThreads), msm, s, p, d.head_size);
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
  if (a->max_pages > nsel && sa->n_top > 0) {
    // pages per CTA: as few as fill the GPU about four times over
    const int cand = a->max_pages - sa->n_sink - sa->n_window;
    const int64_t pairs = (int64_t)a->n_seqs * d.n_kv_heads;
    const int64_t target = std::max<int64_t>(1, (int64_t)c->num_sms * 4 / pairs);
    int per = (int)((cand + target - 1) / target);
    per = std::max(16, (per + 15) / 16 * 16);
    void* args[] = {&p, &per};
    if ((st = launch_pdl_c(score_kernel_for(d), dim3((cand + per - 1) / per, d.n_kv_heads, a->n_seqs),
                           dim3(kScoreThreads), 0, s, args)))
      return st;
  }
  if ((st = pdl_launch(kv_select_kernel, dim3(d.n_kv_heads, a->n_seqs), dim3(kSelThreads), 0, s, p))) return st;
  return kv_attn_launch(kv, *a, p.phys, nsel, c, s);
}

}  // extern "C"
