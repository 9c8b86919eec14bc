// What the sources of gguf_kv_attn_shared share: the line of tiles and a
// CTA's place on it.
#pragma once
#include <math.h>

#include "paged_kv.cuh"
#include "pdl_launch.cuh"

namespace vireo {

constexpr int kShaCtas = 160;  // that the workspace has room for
constexpr float kShaLog2e = 1.4426950408889634f;

struct ShReq {
  int own, page0;     // positions of the request's own, behind so many pages of its row
  int lead, members;  // the first request of its group, or -1 where it takes nothing from it; and their number (1: no group)
  int prefix;         // of a group's first request: positions shared, else 0
  int row0;           // rows of pieces before this request's
  long long line;     // tiles before this request's
};
struct ShParams {
  const void *q, *k, *v;
  void* out;
  int64_t q_stride, out_stride, table_stride, page_stride, head_stride, pos_stride;
  const int32_t *table, *kv_len, *cu, *shared;
  int n_seqs, max_pages, n_pages, n_groups;
  int H, G, R, ps_shift;
  int rt, nsub, tile_shift;  // rows of a unit at most, units of one request's heads, tile
  int ctas;
  float scale;  // times log2(e)
  ShReq* req;   // [n_seqs + ctas] request i as CTA c sees it at i + c: those of the CTA's stretch
  ShReq* all;   // [n_seqs] for the join
  long long* total;
  float* part;  // rows of HS + 4: accumulator, maximum, sum
  int* err;
};

// CTA i takes tiles [at(i), at(i + 1)): q each, the first r of them one more
struct ShCut {
  long long q;
  int r;
  VDEV ShCut(long long total, int ctas) : q(total / ctas), r((int)(total % ctas)) {}
  VDEV long long at(int i) const { return q * i + min(i, r); }
  VDEV int of(long long u) const {  // the CTA that takes tile u
    const long long wide = (q + 1) * r;
    return u < wide ? (int)(u / (q + 1)) : r + (int)((u - wide) / q);
  }
};
VDEV int sh_ctas(const ShParams& p, long long total) { return (int)min((long long)p.ctas, total); }
VDEV int sh_blocks(const ShParams& p, int members) { return (int)(((long long)members * p.R + p.rt - 1) / p.rt); }
VDEV int sh_tiles(const ShParams& p, int len) {
  return (int)(((long long)len + (1 << p.tile_shift) - 1) >> p.tile_shift);
}


// What a CTA keeps while it looks for its stretch (shared memory that the
// kernel uses otherwise afterwards)
constexpr int kShaSeqs = 8192;  // requests, and groups
struct ShPlanned {
  long long red[32], begin, end, line;  // of the stretch; of its first request
  int redi[32], first;
};
inline size_t sh_plan_smem(int n_seqs, int n_groups) {
  return sizeof(ShPlanned) + 4 * ((size_t)n_seqs + 2 * (size_t)n_groups + 1);
}

// a place on the line
struct ShWalk {
  ShReq q;
  int i, own, kh, sub, tile, len, ntile, blocks;
  long long left;
  VDEV void unit(const ShParams& p) {
    len = own ? q.own : q.prefix;
    ntile = sh_tiles(p, len);
    blocks = own ? p.nsub : sh_blocks(p, q.members);
  }
  // tile `at` of a request's tiles
  VDEV void begin(const ShParams& p, int first, long long at, long long count) {
    i = first;
    left = count;
    own = kh = sub = tile = 0;
    if (left <= 0) return;
    q = p.req[i + (int)blockIdx.x];
    int per = q.prefix ? sh_blocks(p, q.members) : 0, nt = sh_tiles(p, q.prefix);
    if (at >= (long long)p.G * per * nt) {
      at -= (long long)p.G * per * nt;
      own = 1;
      per = p.nsub;
      nt = sh_tiles(p, q.own);
    }
    const int x = (int)(at / nt);
    tile = (int)(at - (long long)x * nt);
    kh = x / per;
    sub = x - kh * per;
    unit(p);
  }
  VDEV int count() const { return (int)min((long long)(ntile - tile), left); }  // tiles of the unit that are this CTA's
  VDEV void next(const ShParams& p) {
    left -= count();
    tile = 0;
    if (left <= 0 || ++sub < blocks) return;
    sub = 0;
    if (++kh < p.G) return;
    kh = 0;
    if (!own && q.own > 0) {
      own = 1;
    } else {
      do q = p.req[++i + (int)blockIdx.x];  // left > 0: a request with tiles follows
      while (q.prefix == 0 && q.own == 0);
      own = q.prefix == 0;
    }
    unit(p);
  }
  // the unit's rows: rows row0 .. row0 + rows - 1 of the members' heads of kv head kh, member after member
  VDEV int row0(const ShParams& p) const { return sub * p.rt; }
  VDEV int rows(const ShParams& p) const { return min(p.rt, (own ? 1 : q.members) * p.R - sub * p.rt); }
  // request and head of one of them
  VDEV void row(const ShParams& p, int r, int& seq, int& head) const {
    const int f = row0(p) + r, m = f / p.R;
    seq = i + m;
    head = kh * p.R + f - m * p.R;
  }
  VDEV const int32_t* pages(const ShParams& p) const {  // of the unit's positions
    return p.table + (int64_t)i * p.table_stride + (own ? q.page0 : 0);
  }
  // nothing to join, and (out may be q) no other unit that reads the rows
  VDEV bool whole() const { return own && q.members == 1 && count() == ntile; }
  VDEV int64_t part_row(const ShParams& p) const {
    const int base = own ? q.row0 + (q.prefix ? q.members * p.H : 0) + kh * p.R
                         : q.row0 + kh * q.members * p.R;
    return (int64_t)base + row0(p) + (int64_t)p.rt * blockIdx.x;
  }
};

VDEV float sh_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Finds the CTA's stretch of the line, by all of its NT threads (a multiple of
// 32): lengths and groups to shared memory, a request (or a few neighbouring
// ones) to a thread, prefix sums.  Every CTA computes all of it for itself:
// one read's latency and a few hundred cycles, where a launch ahead of this
// one cost 6 us.
template <int NT>
VDEV ShWalk sh_plan(const ShParams& p, uint8_t* smem) {
  constexpr int NW = NT / 32;
  ShPlanned* sh = reinterpret_cast<ShPlanned*>(smem);
  int* cu = reinterpret_cast<int*>(sh + 1);  // as it is taken
  int* shared = cu + p.n_groups + 1;
  int* len = shared + p.n_groups;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = p.n_seqs, ng = p.n_groups;
  bool bad = false;
  for (int j = tid; j < ng; j += NT) {
    const int s = p.shared[j];
    bad |= s < 0;
    shared[j] = max(s, 0);
  }
  for (int i = tid; i < n; i += NT) {
    const int x = max(p.kv_len[i], 0), top = p.max_pages << p.ps_shift;
    bad |= x > top;
    len[i] = min(x, top);
  }
  // cu, each at least the largest before it
  for (int base = 0, most = 0; base <= ng; base += NT) {
    const int j = base + tid, given = j <= ng ? p.cu[j] : 0;
    int v = min(max(given, 0), n);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v = max(v, u);
    }
    if (ng >= 32) {  // more than a warp's
      __syncthreads();
      if (lane == 31) sh->redi[warp] = v;
      __syncthreads();
      int all = most;
#pragma unroll
      for (int w = 0; w < NW; w++) {
        if (w == warp) v = max(v, all);
        all = max(all, sh->redi[w]);
      }
      most = all;
    }
    if (j <= ng) {
      bad |= v != given;
      cu[j] = v;
    }
  }
  if (bad) set_error(p.err, VIREO_ERR_ARG);
  __syncthreads();
  const auto tiles_rows = [&](int i, ShReq& q, int& rows) {
    q = {len[i], 0, -1, 1, 0, 0, 0};
    int g = -1;  // the last group that begins at or before it
    for (int step = ng > 0 ? 1 << (31 - __clz(ng)) : 0; step; step >>= 1)
      if (g + step < ng && cu[g + step] <= i) g += step;
    rows = p.H;
    long long t = 0;
    if (g >= 0 && i < cu[g + 1]) {
      const int lead = cu[g], m = cu[g + 1] - lead;
      const int s = m > 1 ? min(shared[g], len[lead]) >> p.ps_shift << p.ps_shift : 0;
      if (s > 0) {
        q.members = m;
        if (i == lead) {
          q.prefix = s;
          t = (long long)p.G * sh_blocks(p, m) * sh_tiles(p, s);
          rows += m * p.H;
        }
        if (q.own >= s) {
          q.lead = lead;
          q.own -= s;
          q.page0 = s >> p.ps_shift;
        }
      }
    }
    return t + (long long)p.G * p.nsub * sh_tiles(p, q.own);
  };
  const int per = (n + NT - 1) / NT, lo = min(n, tid * per), hi = min(n, lo + per);
  long long t = 0;
  int rows = 0;
  ShReq q;
  for (int i = lo; i < hi; i++) {
    int r;
    t += tiles_rows(i, q, r);
    rows += r;
  }
  long long ti = t;
  int ri = rows;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, ti, o);
    const int r = __shfl_up_sync(0xffffffffu, ri, o);
    if (lane >= o) {
      ti += u;
      ri += r;
    }
  }
  if (lane == 31) {
    sh->red[warp] = ti;
    sh->redi[warp] = ri;
  }
  __syncthreads();
  long long total = 0;
  int rb = 0;
#pragma unroll 4
  for (int w = 0; w < NW; w++) {
    if (w == warp) {
      ti += total;
      ri += rb;
    }
    total += sh->red[w];
    rb += sh->redi[w];
  }
  const int ctas = sh_ctas(p, total), c = blockIdx.x;
  long long begin = 0, end = 0;
  if (c < ctas) {
    const ShCut cut(total, ctas);
    begin = cut.at(c);
    end = cut.at(c + 1);
  }
  if (c == 0 && tid == 0) *p.total = total;
  long long line = ti - t;
  int row0 = ri - rows;
  for (int i = lo; i < hi; i++) {
    int r;
    const long long mine = tiles_rows(i, q, r);
    q.line = line;
    q.row0 = row0;
    if (line < end && (line >= begin || line + mine > begin)) p.req[i + c] = q;
    if (mine > 0 && line <= begin && begin < line + mine) {
      sh->first = i;
      sh->line = line;
    }
    if (i % gridDim.x == c) p.all[i] = q;
    line += mine;
    row0 += r;
  }
  __syncthreads();
  ShWalk w;
  w.begin(p, sh->first, begin - sh->line, end - begin);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // copies may fill it
  __syncthreads();                                               // the shared memory is free
  return w;
}

// A kernel for a pool: rows of a unit, positions of a tile.
struct ShKernel {
  const void *fn, *merge;
  int threads, smem, rt, tile;
  bool maps;  // takes tensor maps of the pools
};
// 16-bit caches (paged_shared_mma.cu); merge is the caller's
ShKernel sh_mma_kernel(const gguf_kv_desc& d);

}  // namespace vireo
