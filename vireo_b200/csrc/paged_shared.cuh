// What the sources of gguf_kv_attn_shared share: the line of tiles and a
// CTA's place on it.
#pragma once
#include <math.h>

#include "paged_kv.cuh"
#include "pdl_launch.cuh"

namespace vireo {

constexpr int kShaSms = 160;  // that the workspace has room for
constexpr float kShaLog2e = 1.4426950408889634f;

struct ShReq {
  int own, page0;     // positions of the request's own, behind so many pages of its row
  int lead, members;  // the first request of its group, or -1 where it takes nothing from it; and their number (1: no group)
  int prefix;         // of a group's first request: positions shared, else 0
  int row0;           // rows of pieces before this request's
  int line;           // tiles before this request's
};
struct ShParams {
  const void *q, *k, *v;
  void* out;
  int64_t q_stride, out_stride, table_stride, page_stride, head_stride, pos_stride;
  const int32_t *table, *kv_len, *cu, *shared;
  int n_seqs, max_pages, n_pages, n_groups;
  int H, G, R, ps_shift;
  int rt, nsub;              // rows of a unit at most, units of one request's heads
  int rt_shift, tile_shift;  // powers of two: divisions here are latency, 64-bit ones half a microsecond
  int ctas;
  float scale;  // times log2(e)
  struct ShUnit* units;  // CTA c's v-th unit on the line at v + c
  ShReq* all;            // [n_seqs] for the join
  int* total;
  float* part;  // rows of HS + 4: accumulator, maximum, sum
  uint8_t* img;  // rows of q as a kernel wants them, eight at a time
  int8_t* up;    // a value to each of these rows
  struct ShEight* eights;  // whose each eight are
  int* err;
};

// CTA i takes tiles [at(i), at(i + 1)): q each, the first r of them one more.
// The line's length fits an int: the host sees to it.
struct ShCut {
  uint32_t q, r;
  VDEV ShCut(int total, int ctas) : q((uint32_t)total / (uint32_t)ctas), r((uint32_t)total - q * ctas) {}
  VDEV int at(int i) const { return (int)(q * i + min((uint32_t)i, r)); }
  VDEV int of(int u) const {  // the CTA that takes tile u
    const uint32_t wide = (q + 1) * r;
    return (int)((uint32_t)u < wide ? u / (q + 1) : r + (u - wide) / q);
  }
};
VDEV int sh_ctas(const ShParams& p, int total) { return min(p.ctas, total); }
// eight rows of q, or what is left of a unit's: rows row .. of the heads of kv
// head kh, request after request from seq on
struct alignas(16) ShEight {
  int seq, row, n_kh;  // rows and 16 kh
  int fill;            // written in one access of 16 bytes
};
VDEV int sh_blocks(const ShParams& p, int members) { return (members * p.R + p.rt - 1) >> p.rt_shift; }
VDEV int sh_tiles(const ShParams& p, int len) {
  return (int)(((long long)len + (1 << p.tile_shift) - 1) >> p.tile_shift);
}

// A CTA's part of a unit: tiles tile .. tile + count - 1 of its positions, for
// `rows` rows from row0 on of the members' heads of a kv head, member after
// member.  Everyone in the CTA reads the list of them.
struct alignas(16) ShUnit {
  int seq;            // the first member, on whose pages the positions are,
  int page0, len;     // behind so many pages of its row; and their number
  int kh, row0, rows;
  int tile, count;
  int part;           // first row of the piece
  int img;            // first eight rows of q's image
  // request and head of one of the rows
  VDEV void row(const ShParams& p, int r, int& s, int& head) const {
    const int f = row0 + r, m = f / p.R;
    s = seq + m;
    head = kh * p.R + f - m * p.R;
  }
  VDEV const int32_t* pages(const ShParams& p) const { return p.table + (int64_t)seq * p.table_stride + page0; }
};

// What a CTA keeps while it looks for its stretch (shared memory that the
// kernel uses otherwise afterwards)
constexpr int kShaSeqs = 8192;  // requests, and groups
struct ShPlanned {
  int tiles[32], rows[32], units[32], eights[32], first, last, img, end;
};
inline size_t sh_plan_smem(int n_seqs, int n_groups) {
  return sizeof(ShPlanned) + 4 * ((size_t)n_seqs + 2 * (size_t)n_groups + 1);
}

VDEV float sh_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The CTA's units, by all of its NT threads (a multiple of 32): lengths and
// groups to shared memory, a request (or a few neighbouring ones) to a thread,
// prefix sums, and the units that lie in the CTA's stretch.  Every CTA computes
// all of it for itself: one read's latency and some hundred cycles, where a
// launch ahead of this one cost 6 us.
struct ShStretch {
  const ShUnit* units;
  int n, img, eights;  // units; with IMG, of q's images the first eight rows and their number
};
template <int NT, bool IMG>
VDEV ShStretch sh_plan(const ShParams& p, uint8_t* smem) {
  constexpr int NW = NT / 32;
  ShPlanned* sh = reinterpret_cast<ShPlanned*>(smem);
  int* cu = reinterpret_cast<int*>(sh + 1);  // as it is taken
  int* shared = cu + p.n_groups + 1;
  int* len = shared + p.n_groups;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = p.n_seqs, ng = p.n_groups, c = blockIdx.x;
  bool bad = false;
  // the first of each on their way together
  int s0 = tid < ng ? p.shared[tid] : 0, x0 = tid < n ? p.kv_len[tid] : 0, c0 = tid <= ng ? p.cu[tid] : 0;
#pragma unroll 1
  for (int j = tid; j < ng; j += NT) {
    bad |= s0 < 0;
    shared[j] = max(s0, 0);
    if (j + NT < ng) s0 = p.shared[j + NT];
  }
#pragma unroll 1
  for (int i = tid; i < n; i += NT) {
    const int x = max(x0, 0), top = p.max_pages << p.ps_shift;
    bad |= x > top;
    len[i] = min(x, top);
    if (i + NT < n) x0 = p.kv_len[i + NT];
  }
  // cu, each at least the largest before it
#pragma unroll 1
  for (int base = 0, most = 0; base <= ng; base += NT) {
    const int j = base + tid, given = base == 0 ? c0 : j <= ng ? p.cu[j] : 0;
    int v = min(max(given, 0), n);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v = max(v, u);
    }
    if (ng >= 32) {  // more than a warp's
      __syncthreads();
      if (lane == 31) sh->rows[warp] = v;
      __syncthreads();
      int all = most;
#pragma unroll 1
      for (int w = 0; w < NW; w++) {
        if (w == warp) v = max(v, all);
        all = max(all, sh->rows[w]);
      }
      most = all;
    }
    if (j <= ng) {
      bad |= v != given;
      cu[j] = v;
    }
  }
  if (bad) set_error(p.err, VIREO_ERR_ARG);
  if (tid == 0) sh->first = sh->last = sh->img = sh->end = 0;
  __syncthreads();
  struct Share {
    ShReq q;
    int blocks, nts, nto, rows, units, eights, tiles;  // row blocks and tiles of the prefix, tiles of its own
  };
  const auto share_of = [&](int i) {
    Share s;
    s.q = {len[i], 0, -1, 1, 0, 0, 0};
    s.blocks = s.nts = 0;
    s.rows = p.H;
    int g = -1;  // the last group that begins at or before it
    for (int step = ng > 0 ? 1 << (31 - __clz(ng)) : 0; step; step >>= 1)
      if (g + step < ng && cu[g + step] <= i) g += step;
    if (g >= 0 && i < cu[g + 1]) {
      const int lead = cu[g], m = cu[g + 1] - lead;
      const int x = m > 1 ? min(shared[g], len[lead]) >> p.ps_shift << p.ps_shift : 0;
      if (x > 0) {
        s.q.members = m;
        if (i == lead) {
          s.q.prefix = x;
          s.blocks = sh_blocks(p, m);
          s.nts = sh_tiles(p, x);
          s.rows += m * p.H;
        }
        if (s.q.own >= x) {
          s.q.lead = lead;
          s.q.own -= x;
          s.q.page0 = x >> p.ps_shift;
        }
      }
    }
    s.nto = sh_tiles(p, s.q.own);
    s.units = p.G * (s.blocks + (s.nto ? p.nsub : 0));
    // rows eight at a time: a block but the last is of 128.  Only of units that
    // there are: a CTA reads all from its first unit's to its last one's.
    s.eights = IMG ? p.G * ((s.blocks ? (s.q.members * p.R + 7) / 8 : 0) + (s.nto ? (p.R + 7) / 8 : 0)) : 0;
    s.tiles = p.G * (s.blocks * s.nts + p.nsub * s.nto);
    return s;
  };
  const int per = (n + NT - 1) / NT, lo = min(n, tid * per), hi = min(n, lo + per);
  Share s = {};
  int t = 0, rows = 0, units = 0, eights = 0;
#pragma unroll 1
  for (int i = hi - 1; i >= lo; i--) {  // the first is at hand afterwards
    s = share_of(i);
    t += s.tiles;
    rows += s.rows;
    units += s.units;
    eights += s.eights;
  }
  int ti = t, ri = rows, ui = units, ei = eights;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, ti, o), y = __shfl_up_sync(0xffffffffu, ri, o),
              z = __shfl_up_sync(0xffffffffu, ui, o), v = IMG ? __shfl_up_sync(0xffffffffu, ei, o) : 0;
    if (lane >= o) {
      ti += x;
      ri += y;
      ui += z;
      ei += v;
    }
  }
  if (lane == 31) {
    sh->tiles[warp] = ti;
    sh->rows[warp] = ri;
    sh->units[warp] = ui;
    sh->eights[warp] = ei;
  }
  __syncthreads();
  // the warps before this one, and all: a lane each
  const int a = lane < NW ? sh->tiles[lane] : 0;
  const int total = __reduce_add_sync(0xffffffffu, a);
  ti += __reduce_add_sync(0xffffffffu, lane < warp ? a : 0);
  ri += __reduce_add_sync(0xffffffffu, lane < warp ? sh->rows[lane] : 0);
  ui += __reduce_add_sync(0xffffffffu, lane < warp ? sh->units[lane] : 0);
  if (IMG) ei += __reduce_add_sync(0xffffffffu, lane < warp ? sh->eights[lane] : 0);
  const int ctas = sh_ctas(p, total);
  int begin = 0, end = 0;
  if (c < ctas) {
    const ShCut cut(total, ctas);
    begin = cut.at(c);
    end = cut.at(c + 1);
  }
  if (c == 0 && tid == 0) *p.total = total;
  int line = ti - t, row0 = ri - rows, unit0 = ui - units, eight0 = ei - eights;
#pragma unroll 1
  for (int i = lo; i < hi; i++) {
    if (i > lo) s = share_of(i);
    s.q.line = line;
    s.q.row0 = row0;
    if (i % gridDim.x == c) p.all[i] = s.q;
    // the prefix's units, then its own
    int at = line, unit = unit0, part = row0, eight = eight0;
#pragma unroll 1
    for (int own = 0; own < 2; own++) {
      const int nt = own ? s.nto : s.nts, blocks = own ? p.nsub : s.blocks, m = own ? 1 : s.q.members;
      const int count = nt ? p.G * blocks : 0, stop = at + count * nt;
      if (count && at < end && stop > begin) {
#pragma unroll 1
        for (int k = begin > at ? (begin - at) / nt : 0; k < count; k++) {
          const int a = at + k * nt, from = max(a, begin), to = min(a + nt, end);
          if (from >= to) break;
          const int kh = k / blocks, sub = k - kh * blocks;
          ShUnit u;
          u.seq = i;
          u.page0 = own ? s.q.page0 : 0;
          u.len = own ? s.q.own : s.q.prefix;
          u.kh = kh;
          u.row0 = sub * p.rt;
          u.rows = min(p.rt, m * p.R - u.row0);
          u.tile = from - a;
          u.count = to - from;
          u.part = part + kh * m * p.R + u.row0 + p.rt * c;
          u.img = eight + kh * ((m * p.R + 7) / 8) + u.row0 / 8 + 16 * c;
          p.units[unit + k + c] = u;
          if (from == begin) {
            sh->first = unit + k;
            sh->img = u.img;
          }
          const int next = u.img + (u.rows + 7) / 8;
          if (to == end) {
            sh->last = unit + k + 1;
            sh->end = next;
          }
          if constexpr (IMG)
            for (int x = u.img; x < next; x++) {
              const int j = x - u.img;
              p.eights[x] = {i, u.row0 + 8 * j, max(0, min(8, u.rows - 8 * j)) | kh << 4, 0};
            }
        }
      }
      at = stop;
      unit += count;
      if (!own && s.q.prefix) {
        part += m * p.H;
        eight += p.G * ((m * p.R + 7) / 8);
      }
    }
    line += s.tiles;
    row0 += s.rows;
    unit0 += s.units;
    eight0 += s.eights;
  }
  __syncthreads();
  const ShStretch got = {p.units + sh->first + c, end > begin ? sh->last - sh->first : 0, sh->img,
                         sh->end - sh->img};
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // copies may fill it
  __syncthreads();                                               // the shared memory is free
  return got;
}

// A kernel for a pool: rows of a unit, positions of a tile.
struct ShKernel {
  const void* fn;
  int threads, smem, rt, tile;
  bool maps;  // takes tensor maps of the pools
  int img;    // bytes of eight rows' image
  int per_sm; // CTAs
};
// 16-bit caches (paged_shared_mma.cu)
ShKernel sh_mma_kernel(const gguf_kv_desc& d);

}  // namespace vireo
