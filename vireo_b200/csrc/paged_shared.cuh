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
struct ShStart {
  int i, own, kh, sub, tile, ctas;
  long long left;
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
  int* cu_s;    // [n_groups + 1] cu as it is taken
  ShReq* req;   // [n_seqs]
  ShStart* start;  // [ctas]
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
  VDEV void begin(const ShParams& p) {
    const ShStart s = p.start[blockIdx.x];
    i = s.i;
    own = s.own;
    kh = s.kh;
    sub = s.sub;
    tile = s.tile;
    left = s.left;
    if (left > 0) {
      q = p.req[i];
      unit(p);
    }
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
      do q = p.req[++i];  // left > 0: a request with tiles follows
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

// A kernel for a pool: rows of a unit, positions of a tile.
struct ShKernel {
  const void *fn, *merge;
  int threads, smem, rt, tile;
  bool maps;  // takes tensor maps of the pools
};
// 16-bit caches (paged_shared_mma.cu); merge is the caller's
ShKernel sh_mma_kernel(const gguf_kv_desc& d);

}  // namespace vireo
