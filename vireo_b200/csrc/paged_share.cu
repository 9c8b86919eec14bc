// Pages that requests hold together (include/gguf_kv.h): rows of the block
// table that continue other rows, the copies that go with them, and the
// compaction of a pool.
#include <string.h>

#include "paged_kv.cuh"
#include "pdl_launch.cuh"

namespace vireo {

constexpr int kShThreads = 512, kShWarps = kShThreads / 32;
constexpr int kShMaxSeqs = 8192;
constexpr int kShCluster = 8;
constexpr int kShChunk = 128;  // table entries that a warp takes at once

// Every phase of these calls reads what all of the one before has written.
// Where one cluster of CTAs is enough for the work, its barrier stands between
// the phases of a single launch; else every phase is a launch of its own.
// Integers throughout, and everything has one place: the order in which
// atomics arrive shows nowhere.
enum SharePart { kShAll, kShFirst, kShSecond, kShThird, kShFourth };

VDEV void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n barrier.cluster.wait.aligned;" ::: "memory");
}

VDEV int pages_of(int len, int ps_shift) { return (int)(((long long)len + (1 << ps_shift) - 1) >> ps_shift); }
// a row has 2^this chunks, some of them behind its end: a division would be latency
VDEV int chunk_shift(int max_pages) {
  const int chunks = (max_pages + kShChunk - 1) / kShChunk;
  return chunks > 1 ? 32 - __clz(chunks - 1) : 0;
}
// a place in the ring, from one less than twice its length
VDEV unsigned int in_ring(unsigned int x, unsigned int np) { return x >= np ? x - np : x; }
VDEV int row_len(const int32_t* kv_len, int i, int most, int* err) {
  const int n = max(kv_len[i], 0);
  if (n > most) {
    set_error(err, VIREO_ERR_ARG);
    return most;
  }
  return n;
}

// exclusive sum over the block; tot: the block's
VDEV int block_sum(int v, int* red, int& tot) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  __syncthreads();  // red may still be read from the previous sum
  if (lane == 31) red[warp] = inc;
  __syncthreads();
  int before = 0;
  tot = 0;
#pragma unroll
  for (int w = 0; w < kShWarps; w++) {
    const int x = red[w];
    if (w < warp) before += x;
    tot += x;
  }
  return before + inc - v;
}

// ---------------------------------------------------------------------------
// Rows that continue other rows.
//
// First, by one CTA: per row what it keeps, whether its unfinished page stays
// or is copied, and with prefix sums who gets a page for the copy.  Of a
// parent's children only those that end in the last page that any of them
// reaches can keep theirs (for the others some child holds all of it), and of
// those the first; so a maximum and a minimum per parent decide.  The child
// with the most of the parent's pages is its heir, and the two cancel: holders
// are counted for the other children's pages (one more) and for what is left
// of the parent's (one less), so that rows that merely go on cost no atomics.
//
// Second: table entries and holders, a warp to 128 entries.  Third: the pages
// whose holders ran out, in rising order, a stretch of pages to a warp.
//
// Latency-bound: three phases of a few dependent loads each (64 rows of 63 pages
// 9.3 us, 512 rows of up to 63 13.7, floor below 2).
// ---------------------------------------------------------------------------
struct ForkParams {
  gguf_kv_fork_args a;
  int ps_shift;
  SharePart part;
  int* taken;  // [n_out] pages of the parent's that the row holds; the heir's with kHeir
  int* heir;   // [n_seqs] pages that the heir holds
  int* note;   // head, count, pages granted; then per CTA the pages let go
  int* err;
};
constexpr unsigned int kHeir = 0x80000000u;
constexpr int kNotes = 16;

static size_t fork_smem(int n_seqs, int n_out) { return (size_t)n_seqs * 16 + (size_t)n_out * 8; }

VDEV void fork_rows(const ForkParams& p) {
  extern __shared__ __align__(16) uint8_t shared[];
  __shared__ int red[kShWarps];
  const gguf_kv_fork_args& a = p.a;
  const int tid = threadIdx.x, ns = a.n_seqs, no = a.n_out, most = a.max_pages << p.ps_shift;
  unsigned long long* key = reinterpret_cast<unsigned long long*>(shared);  // [ns] the heir: most pages, then first
  int* longest = reinterpret_cast<int*>(key + ns);                          // [ns] positions of the longest child
  int* first = longest + ns;                                                // [ns] first child in its last page
  int* want = first + ns;                                                   // [no]
  int* par = want + no;                                                     // [no]
  const unsigned int np = (unsigned int)a.n_pages, head = (unsigned int)a.state[0] % np;
  const int count = min(max(a.state[1], 0), a.n_pages);
  for (int i = tid; i < ns; i += kShThreads) {
    key[i] = 0;
    longest[i] = 0;
    first[i] = INT32_MAX;
  }
  __syncthreads();
  for (int i = tid; i < no; i += kShThreads) {
    int q = a.parent[i];
    if (q < -1 || q >= ns) {
      set_error(p.err, VIREO_ERR_ARG);
      q = -1;
    }
    int w = 0;
    if (q >= 0) {
      w = row_len(a.kv_len, q, most, p.err);
      if (a.keep && a.keep[i] >= 0) w = min(w, a.keep[i]);
      atomicMax(&longest[q], w);
    }
    par[i] = q;
    want[i] = w;
  }
  __syncthreads();
  for (int i = tid; i < no; i += kShThreads) {
    const int q = par[i];
    if (q >= 0 && want[i] > (longest[q] >> p.ps_shift << p.ps_shift)) atomicMin(&first[q], i);
  }
  __syncthreads();
  int used = 0;
  for (int base = 0; base < no; base += kShThreads) {
    const int i = base + tid, q = i < no ? par[i] : -1;
    const int w = i < no ? want[i] : 0, whole = w >> p.ps_shift, tail = w & ((1 << p.ps_shift) - 1);
    bool stays = false;
    int last = -1;
    if (tail) {
      last = a.table[(int64_t)q * a.table_stride + whole];
      stays = first[q] == i && (last < 0 || last >= a.n_pages || a.shares[last] == 0);
    }
    int tot;
    const bool need = tail && !stays;
    const int rank = used + block_sum(need, red, tot);
    const bool granted = !need || rank < count;
    if (i < no) {
      const bool copied = need && granted;
      const int taken = granted ? whole + stays : 0;
      a.kv_len_out[i] = granted ? w : 0;
      a.granted[i] = granted;
      a.src[i] = copied ? last : -1;
      a.dst[i] = copied ? a.ring[in_ring(head + (unsigned int)rank, np)] : -1;
      a.rows[i] = copied ? tail : 0;
      if (q >= 0 && granted) atomicMax(&key[q], (unsigned long long)(taken + 1) << 32 | (uint32_t)~i);
      want[i] = taken;
    }
    used = min(used + tot, count);
  }
  __syncthreads();
  for (int i = tid; i < ns; i += kShThreads) p.heir[i] = key[i] ? (int)(key[i] >> 32) - 1 : 0;
  for (int i = tid; i < no; i += kShThreads) {
    const bool is = par[i] >= 0 && key[par[i]] && (uint32_t)key[par[i]] == (uint32_t)~i;
    p.taken[i] = want[i] | (is ? kHeir : 0u);
  }
  if (tid == 0) {
    p.note[0] = (int)head;
    p.note[1] = count;
    p.note[2] = used;
  }
}

// A warp reads what 32 of its items are at once, a lane each, and then has four
// items' entries on their way: one after the other, every item waited for two
// reads of its own.
VDEV void fork_entries(const ForkParams& p) {
  const gguf_kv_fork_args& a = p.a;
  constexpr int E = kShChunk / 32, U = 4;
  const int lane = threadIdx.x & 31, warp = blockIdx.x * kShWarps + (threadIdx.x >> 5), nw = gridDim.x * kShWarps;
  const int shift = chunk_shift(a.max_pages), most = a.max_pages << p.ps_shift;
  const int64_t items = (int64_t)(a.n_out + a.n_seqs) << shift;
  for (int64_t it0 = warp; it0 < items; it0 += 32ll * nw) {
    const int64_t it = it0 + (int64_t)lane * nw;
    // this lane's item: entries first .. n - 1 of row `from`; of a new row they go
    // to row `to`, of an old one they are let go from `kept` on
    int from = 0, to = -1, first = 0, n = 0, kept = 0, last = 0, tail = 0;
    if (it < items) {
      const int row = (int)(it >> shift);
      first = ((int)it & ((1 << shift) - 1)) * kShChunk;
      if (row < a.n_out) {
        const unsigned int t = (unsigned int)p.taken[row];
        to = row;
        n = (int)(t & ~kHeir);
        kept = t & kHeir ? 1 : 0;
        tail = a.rows[row] > 0;
        last = a.dst[row];
        from = max(a.parent[row], 0);
      } else {
        from = row - a.n_out;
        n = pages_of(row_len(a.kv_len, from, most, p.err), p.ps_shift);
        kept = p.heir[from];
      }
    }
    unsigned int work = __ballot_sync(0xffffffffu, first < n + tail);
    while (work) {
      int src[U], id[U][E];
#pragma unroll
      for (int u = 0; u < U; u++) {
        src[u] = work ? __ffs(work) - 1 : -1;
        work &= work - 1;
        const int s = max(src[u], 0), f = __shfl_sync(0xffffffffu, from, s), j0 = __shfl_sync(0xffffffffu, first, s),
                  m = __shfl_sync(0xffffffffu, n, s);
        const int32_t* row = a.table + (int64_t)f * a.table_stride;
#pragma unroll
        for (int e = 0; e < E; e++) {
          const int j = j0 + 32 * e + lane;
          id[u][e] = src[u] >= 0 && j < m ? row[j] : 0;
        }
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int s = max(src[u], 0), j0 = __shfl_sync(0xffffffffu, first, s), m = __shfl_sync(0xffffffffu, n, s),
                  t = __shfl_sync(0xffffffffu, to, s), k = __shfl_sync(0xffffffffu, kept, s),
                  more = __shfl_sync(0xffffffffu, tail, s), fresh = __shfl_sync(0xffffffffu, last, s);
        if (src[u] < 0) continue;
#pragma unroll
        for (int e = 0; e < E; e++) {
          const int j = j0 + 32 * e + lane, x = id[u][e];
          const bool inside = x >= 0 && x < a.n_pages;
          if (t >= 0) {
            if (j < m) {
              a.table_out[(int64_t)t * a.table_out_stride + j] = x;
              if (!k && inside) atomicAdd(&a.shares_out[x], 1);
            } else if (j == m && more) {
              a.table_out[(int64_t)t * a.table_out_stride + j] = fresh;
            }
          } else if (j < m) {
            if (!inside)
              set_error(p.err, VIREO_ERR_ARG);
            else if (j >= k)
              atomicAdd(&a.shares_out[x], -1);
          }
        }
      }
    }
  }
}

// pages without holders: a stretch of pages per warp of one cluster
VDEV void fork_free(const ForkParams& p) {
  __shared__ int red[kShWarps];
  const gguf_kv_fork_args& a = p.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nw = gridDim.x * kShWarps, per = ((a.n_pages + nw - 1) / nw + 31) / 32 * 32;
  const int64_t lo = (int64_t)(blockIdx.x * kShWarps + warp) * per;
  const int p0 = (int)min((int64_t)a.n_pages, lo), p1 = (int)min((int64_t)a.n_pages, lo + per);
  int mine = 0;
#pragma unroll 8
  for (int i = p0; i < p1; i += 32)
    mine += __popc(__ballot_sync(0xffffffffu, i + lane < p1 && a.shares_out[i + lane] < 0));
  int tot;
  int at = block_sum(lane == 0 ? mine : 0, red, tot);
  at = __shfl_sync(0xffffffffu, at, 0);
  if (threadIdx.x == 0) p.note[3 + blockIdx.x] = tot;
  cluster_sync();
  int all = 0;
  for (int c = 0; c < (int)gridDim.x; c++) {
    const int x = p.note[3 + c];
    if (c < (int)blockIdx.x) at += x;
    all += x;
  }
  const unsigned int np = (unsigned int)a.n_pages, head = (unsigned int)p.note[0];
  const int count = p.note[1], used = p.note[2], room = a.n_pages - count;
  if (mine)
    for (int i = p0; i < p1; i += 32) {
      const int s = i + lane < p1 ? a.shares_out[i + lane] : 0;
      const unsigned int gone = __ballot_sync(0xffffffffu, s < 0);
      if (s < 0) {
        const int r = at + __popc(gone & ((1u << lane) - 1u));
        if (s < -1) set_error(p.err, VIREO_ERR_ARG);
        a.shares_out[i + lane] = 0;
        if (r < room) a.ring[in_ring(head + (unsigned int)(count + r), np)] = i + lane;
      }
      at += __popc(gone);
    }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    if (all > room) set_error(p.err, VIREO_ERR_ARG);
    a.state_out[0] = (int)in_ring(head + (unsigned int)used, np);
    a.state_out[1] = count - used + min(all, room);
  }
}

__global__ void __launch_bounds__(kShThreads) kv_fork_kernel(const __grid_constant__ ForkParams p) {
  pdl_launch_dependents();
  pdl_wait();
  if (p.part == kShAll || p.part == kShFirst) {
    if (blockIdx.x == 0) fork_rows(p);
    if (p.a.shares_out != p.a.shares) {
      // the first CTA has its rows; alone it does both
      const int others = gridDim.x > 1 ? (int)gridDim.x - 1 : 1, me = gridDim.x > 1 ? (int)blockIdx.x - 1 : 0;
      if (me >= 0)
#pragma unroll 4
        for (int i = me * kShThreads + threadIdx.x; i < p.a.n_pages; i += others * kShThreads)
          p.a.shares_out[i] = p.a.shares[i];
    }
  }
  if (p.part == kShAll) cluster_sync();
  if (p.part == kShAll || p.part == kShSecond) fork_entries(p);
  if (p.part == kShAll) cluster_sync();
  if (p.part == kShAll || p.part == kShThird) fork_free(p);
}

// ---------------------------------------------------------------------------
// Compaction: a bit per page in use; their prefix sums give every page its
// rank, and with the number m of pages in use and the number of moves follow
// the list, the ring and every page's new number in closed form.  Latency-bound:
// four phases (6 rows 10.6 us, 128 rows of 64 pages 13.6).
// ---------------------------------------------------------------------------
struct CompactParams {
  gguf_kv_compact_args a;
  int ps_shift;
  SharePart part;
  uint32_t* bits;  // [words] pages in use
  int* rank;       // [words] pages in use before the word
  int* note;       // m, moves; then per CTA the pages in use
  int* err;
};

template <class F>
VDEV void compact_entries(const CompactParams& p, F&& f) {
  const gguf_kv_compact_args& a = p.a;
  constexpr int E = kShChunk / 32, U = 4;
  const int lane = threadIdx.x & 31, warp = blockIdx.x * kShWarps + (threadIdx.x >> 5), nw = gridDim.x * kShWarps;
  const int shift = chunk_shift(a.max_pages), most = a.max_pages << p.ps_shift;
  const int64_t items = (int64_t)a.n_seqs << shift;
  for (int64_t it0 = warp; it0 < items; it0 += 32ll * nw) {  // as fork_entries
    const int64_t it = it0 + (int64_t)lane * nw;
    int row = 0, first = 0, n = 0;
    if (it < items) {
      row = (int)(it >> shift);
      first = ((int)it & ((1 << shift) - 1)) * kShChunk;
      n = pages_of(row_len(a.kv_len, row, most, p.err), p.ps_shift);
    }
    unsigned int work = __ballot_sync(0xffffffffu, first < n);
    while (work) {
      int at[U], j0[U], m[U], id[U][E];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int s = work ? __ffs(work) - 1 : 0, has = work != 0;
        work &= work - 1;
        at[u] = __shfl_sync(0xffffffffu, row, s);
        j0[u] = __shfl_sync(0xffffffffu, first, s);
        m[u] = __shfl_sync(0xffffffffu, n, s);
        if (!has) m[u] = 0;
#pragma unroll
        for (int e = 0; e < E; e++) {
          const int j = j0[u] + 32 * e + lane;
          id[u][e] = j < m[u] ? a.table[(int64_t)at[u] * a.table_stride + j] : 0;
        }
      }
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < E; e++) {
          const int j = j0[u] + 32 * e + lane;
          if (j < m[u]) f(at[u], j, id[u][e]);
        }
    }
  }
}

VDEV void compact_ranks(const CompactParams& p) {
  __shared__ int red[kShWarps];
  const gguf_kv_compact_args& a = p.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nw = gridDim.x * kShWarps, words = (a.n_pages + 31) / 32, per = (words + nw - 1) / nw;
  const int w0 = min(words, (blockIdx.x * kShWarps + warp) * per), w1 = min(words, w0 + per);
  int mine = 0;
#pragma unroll 4
  for (int w = w0 + lane; w < w1; w += 32) mine += __popc(p.bits[w]);
#pragma unroll
  for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  int tot;
  int at = block_sum(lane == 0 ? mine : 0, red, tot);
  at = __shfl_sync(0xffffffffu, at, 0);
  if (threadIdx.x == 0) p.note[2 + blockIdx.x] = tot;
  cluster_sync();
  int m = 0;
  for (int c = 0; c < (int)gridDim.x; c++) {
    const int x = p.note[2 + c];
    if (c < (int)blockIdx.x) at += x;
    m += x;
  }
  for (int w = w0, r = at; w < w1; w += 32) {  // ranks of the words, 32 at a time
    const int c = w + lane < w1 ? __popc(p.bits[w + lane]) : 0;
    int inc = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    if (w + lane < w1) {
      p.rank[w + lane] = r + inc - c;
      if (w + lane == m >> 5 || (m == a.n_pages && w + lane == words - 1)) {
        // pages in use below m, and so the free ones there: as many as lie behind
        const unsigned int below = m == a.n_pages ? p.bits[w + lane] : p.bits[w + lane] & ((1u << (m & 31)) - 1u);
        p.note[0] = m;
        p.note[1] = min(m - (r + inc - c + __popc(below)), a.n_copies);
      }
    }
    r += __shfl_sync(0xffffffffu, inc, 31);
  }
  cluster_sync();
  const int moves = p.note[1];
#pragma unroll 4
  for (int w = w0; w < w1; w++) {
    const unsigned int bits = p.bits[w];
    const int id = 32 * w + lane;
    if (id < a.n_pages) {
      const int u = p.rank[w] + __popc(bits & ((1u << lane) - 1u)), f = id - u;  // before it: in use, and free
      const bool used = bits >> lane & 1u, goes = used && u >= m - moves, gets = !used && f < moves;
      if (goes) a.src[u - (m - moves)] = id;
      if (gets) a.dst[f] = id;
      if ((!used && !gets) || goes) a.ring[max(0, f - moves) + max(0, u - (m - moves))] = id;
      if (a.shares_out != a.shares && !goes && !gets) a.shares_out[id] = a.shares[id];
    }
  }
  for (int j = moves + blockIdx.x * kShThreads + threadIdx.x; j < a.n_copies; j += gridDim.x * kShThreads)
    a.src[j] = a.dst[j] = -1;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.state_out[0] = 0;
    a.state_out[1] = a.n_pages - m;
  }
}

__global__ void __launch_bounds__(kShThreads) kv_compact_kernel(const __grid_constant__ CompactParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const gguf_kv_compact_args& a = p.a;
  if (p.part == kShAll || p.part == kShFirst)
    for (int w = blockIdx.x * kShThreads + threadIdx.x; w < (a.n_pages + 31) / 32; w += gridDim.x * kShThreads)
      p.bits[w] = 0;
  if (p.part == kShAll) cluster_sync();
  if (p.part == kShAll || p.part == kShSecond)
    compact_entries(p, [&](int, int, int id) {
      if (id < 0 || id >= a.n_pages)
        set_error(p.err, VIREO_ERR_ARG);
      else
        atomicOr(&p.bits[id >> 5], 1u << (id & 31));
    });
  if (p.part == kShAll) cluster_sync();
  if (p.part == kShAll || p.part == kShThird) compact_ranks(p);
  if (p.part == kShAll) cluster_sync();
  if (p.part == kShAll || p.part == kShFourth) {
    const int m = p.note[0], moves = p.note[1];
    compact_entries(p, [&](int row, int j, int id) {
      if (id >= 0 && id < a.n_pages) {
        const int u = p.rank[id >> 5] + __popc(p.bits[id >> 5] & ((1u << (id & 31)) - 1u));
        if (u >= m - moves) id = a.dst[u - (m - moves)];
      }
      a.table_out[(int64_t)row * a.table_out_stride + j] = id;
    });
    if (a.shares)
      for (int j = blockIdx.x * kShThreads + threadIdx.x; j < moves; j += gridDim.x * kShThreads) {
        const int s = a.src[j], x = a.shares[s];
        a.shares_out[s] = 0;
        a.shares_out[a.dst[j]] = x;
      }
  }
}

// ---------------------------------------------------------------------------
// Pages to pages: a group of threads per pair and pool, 16 bytes at a time.
// Bound by HBM: 891 MB in 141.5 us, 6.3 TB/s; a step's 10.5 MB, in L2, 6.9 us.
// ---------------------------------------------------------------------------
constexpr int kCopyThreads = 256, kCopyLayers = 64;
struct CopyParams {
  const int32_t *src, *dst, *rows;
  int n, n_pages, page, G;
  int chunk_shift;  // 16-byte chunks of a row: a power of two
  int group;        // threads per pair
  int heads_out;    // heads outside positions
  int stream;       // more than L2 holds: past it
  int64_t page_bytes, head_bytes, pos_bytes;
  int* err;
  uint8_t *k[kCopyLayers], *v[kCopyLayers], *means[kCopyLayers];
};

__global__ void __launch_bounds__(kCopyThreads) kv_copy_kernel(const __grid_constant__ CopyParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int i = blockIdx.x * (kCopyThreads / p.group) + threadIdx.x / p.group, t = threadIdx.x % p.group;
  if (i >= p.n) return;
  const int src = p.src[i], dst = p.dst[i], rows = p.rows ? min(p.rows[i], p.page) : p.page;
  if (src < 0 || src == dst) return;
  if (src >= p.n_pages || dst < 0 || dst >= p.n_pages) {
    if (t == 0) set_error(p.err, VIREO_ERR_ARG);
    return;
  }
  const int layer = blockIdx.y >> 1;
  uint8_t* pool = blockIdx.y & 1 ? p.v[layer] : p.k[layer];
  const uint8_t* from = pool + src * p.page_bytes;
  uint8_t* to = pool + dst * p.page_bytes;
  const int inner = p.heads_out ? rows : p.G, total = max(rows, 0) * p.G << p.chunk_shift;
  const int64_t out_bytes = p.heads_out ? p.head_bytes : p.pos_bytes, in_bytes = p.heads_out ? p.pos_bytes : p.head_bytes;
  constexpr int U = 8;
  for (int u0 = t; u0 < total; u0 += U * p.group) {
    uint4 x[U];
    int64_t at[U];
#pragma unroll
    for (int e = 0; e < U; e++) {
      const int u = u0 + e * p.group, r = u >> p.chunk_shift, o = r / inner;
      at[e] = o * out_bytes + (r - o * inner) * in_bytes + (int64_t)(u & ((1 << p.chunk_shift) - 1)) * 16;
      if (u < total) {
        const uint4* q = reinterpret_cast<const uint4*>(from + at[e]);
        x[e] = p.stream ? __ldcs(q) : *q;
      }
    }
#pragma unroll
    for (int e = 0; e < U; e++)
      if (u0 + e * p.group < total) {
        uint4* q = reinterpret_cast<uint4*>(to + at[e]);
        if (p.stream)
          __stcs(q, x[e]);
        else
          *q = x[e];
      }
  }
  if (!(blockIdx.y & 1) && p.means[layer]) {
    const int64_t bytes = (int64_t)p.G << (p.chunk_shift + 4);
    for (int64_t b = 16 * t; b < bytes; b += 16 * p.group)
      *reinterpret_cast<uint4*>(p.means[layer] + dst * bytes + b) =
          *reinterpret_cast<const uint4*>(p.means[layer] + src * bytes + b);
  }
}

static int log2_of(int v) {
  int s = 0;
  while ((1 << s) < v) s++;
  return s;
}

// Phases in one cluster, or launch by launch where a thread of the cluster would
// have more than four items (512 rows of up to 63 pages: 13.7 us in three
// launches, 16 in one; 64 rows 9.3 in one, three launches cost 5 before they
// do anything).
constexpr int64_t kShItems = (int64_t)kShCluster * kShThreads * 4;

template <class P>
static int share_launch(void (*kernel)(P), P& p, int parts, const int* ctas, int one, size_t smem, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kShThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  for (int i = 0; i < (one ? 1 : parts); i++) {
    p.part = one ? kShAll : (SharePart)(kShFirst + i);
    cfg.gridDim = dim3(one ? one : ctas[i]);
    attr[1].val.clusterDim.x = one ? one : i == 2 ? ctas[i] : 1;  // the third phase is of one cluster
    cfg.dynamicSmemBytes = i == 0 ? smem : 0;
    const int st = cuda_status(cudaLaunchKernelEx(&cfg, kernel, p));
    if (st) return st;
  }
  return VIREO_OK;
}

static int cluster_of(int64_t items) {
  const int64_t want = (items + 4 * kShThreads - 1) / (4 * kShThreads);
  return want <= 1 ? 1 : want <= 2 ? 2 : want <= 4 ? 4 : kShCluster;
}
static int grid_of(int64_t items, int num_sms) {
  return (int)std::max<int64_t>(1, std::min<int64_t>(4 * num_sms, (items + kShThreads - 1) / kShThreads));
}
static size_t share_up(size_t v) { return (v + 255) & ~(size_t)255; }
static int page_status(int n_pages, int max_pages, int page_size) {
  if (n_pages < 1 || max_pages < 1 || page_size < 1 || (int64_t)max_pages * page_size > INT32_MAX) return VIREO_ERR_ARG;
  return n_pages > 1 << 30 || page_size < 8 || page_size > 1024 || (page_size & (page_size - 1))
             ? VIREO_ERR_UNSUPPORTED
             : VIREO_OK;
}

}  // namespace vireo

using namespace vireo;

extern "C" {

size_t gguf_kv_fork_workspace(int n_seqs, int n_out) {
  if (n_seqs < 0 || n_out < 0 || n_seqs > kShMaxSeqs || n_out > kShMaxSeqs) return 0;
  return share_up((size_t)n_out * 4) + share_up((size_t)n_seqs * 4) + share_up(kNotes * 4);
}

int gguf_kv_fork(const gguf_kv_fork_args* a, void* stream) {
  if (!a || a->n_seqs < 0 || a->n_out < 0) return VIREO_ERR_ARG;
  int st = page_status(a->n_pages, a->max_pages, a->page_size);
  if (st) return st;
  if (a->n_seqs > kShMaxSeqs || a->n_out > kShMaxSeqs) return VIREO_ERR_UNSUPPORTED;
  if (!a->shares || !a->shares_out || !a->ring || !a->state || !a->state_out || !a->ws || !kv_aligned(a->ws, 256) ||
      a->ws_bytes < gguf_kv_fork_workspace(a->n_seqs, a->n_out) ||
      (a->n_seqs > 0 && (!a->kv_len || !a->table || a->table_stride < a->max_pages)) ||
      (a->n_out > 0 && (!a->parent || !a->table_out || a->table_out_stride < a->max_pages || !a->kv_len_out ||
                        !a->granted || !a->src || !a->dst || !a->rows)) ||
      (a->n_seqs > 0 && a->n_out > 0 && (a->table_out == a->table || a->kv_len_out == a->kv_len)))
    return VIREO_ERR_ARG;
  Ctx* c = ctx_get(&st);
  if (!c) return st;
  DeviceGuard dg(c->device);
  if (dg.status) return dg.status;
  ForkParams p;
  p.a = *a;
  p.ps_shift = log2_of(a->page_size);
  p.taken = (int*)a->ws;
  p.heir = (int*)((uint8_t*)a->ws + share_up((size_t)a->n_out * 4));
  p.note = (int*)((uint8_t*)p.heir + share_up((size_t)a->n_seqs * 4));
  p.err = c->d_err;
  const int64_t entries = (int64_t)(a->n_seqs + a->n_out) * ((a->max_pages + kShChunk - 1) / kShChunk) * 32;
  const int64_t pages = (a->n_pages + 3) / 4, items = std::max(entries, pages);
  const size_t smem = fork_smem(a->n_seqs, a->n_out);
  if (smem > 47 * 1024 &&
      (st = cuda_status(cudaFuncSetAttribute(kv_fork_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)fork_smem(kShMaxSeqs, kShMaxSeqs)))))
    return st;
  const int ctas[3] = {grid_of(a->shares == a->shares_out ? 1 : pages, c->num_sms), grid_of(entries, c->num_sms),
                       cluster_of(pages)};
  return share_launch(kv_fork_kernel, p, 3, ctas, items <= kShItems ? cluster_of(items) : 0, smem,
                      stream ? (cudaStream_t)stream : c->stream);
}

size_t gguf_kv_compact_workspace(int n_pages) {
  if (n_pages < 1) return 0;
  return 2 * share_up(((size_t)n_pages + 31) / 32 * 4) + share_up(kNotes * 4);
}

int gguf_kv_compact(const gguf_kv_compact_args* a, void* stream) {
  if (!a || a->n_seqs < 0 || a->n_copies < 0) return VIREO_ERR_ARG;
  int st = page_status(a->n_pages, a->max_pages, a->page_size);
  if (st) return st;
  if (a->n_seqs > kShMaxSeqs) return VIREO_ERR_UNSUPPORTED;
  if (!a->ring || !a->state_out || !a->ws || !kv_aligned(a->ws, 256) ||
      a->ws_bytes < gguf_kv_compact_workspace(a->n_pages) || !a->shares != !a->shares_out ||
      (a->n_copies > 0 && (!a->src || !a->dst)) ||
      (a->n_seqs > 0 && (!a->kv_len || !a->table || !a->table_out || a->table_stride < a->max_pages ||
                         a->table_out_stride < a->max_pages)) ||
      (a->n_seqs > 1 && a->table_out == a->table && a->table_out_stride != a->table_stride))
    return VIREO_ERR_ARG;
  Ctx* c = ctx_get(&st);
  if (!c) return st;
  DeviceGuard dg(c->device);
  if (dg.status) return dg.status;
  CompactParams p;
  p.a = *a;
  p.ps_shift = log2_of(a->page_size);
  p.bits = (uint32_t*)a->ws;
  const size_t words = share_up(((size_t)a->n_pages + 31) / 32 * 4);
  p.rank = (int*)((uint8_t*)a->ws + words);
  p.note = (int*)((uint8_t*)a->ws + 2 * words);
  p.err = c->d_err;
  const int64_t entries = (int64_t)a->n_seqs * ((a->max_pages + kShChunk - 1) / kShChunk) * 32, pages = a->n_pages;
  const int64_t items = std::max(entries, pages);
  const int ctas[4] = {grid_of(pages / 32, c->num_sms), grid_of(entries, c->num_sms), cluster_of(pages),
                       grid_of(std::max<int64_t>(entries, a->shares ? a->n_copies : 0), c->num_sms)};
  return share_launch(kv_compact_kernel, p, 4, ctas, items <= kShItems ? cluster_of(items) : 0, 0,
                      stream ? (cudaStream_t)stream : c->stream);
}

int gguf_kv_copy(const gguf_kv_copy_args* a, void* stream) {
  if (!a || a->n < 0 || a->n_kv < 0 || (a->n_kv > 0 && !a->kv) || (a->n > 0 && (!a->src || !a->dst)))
    return VIREO_ERR_ARG;
  for (int i = 0; i < a->n_kv; i++) {
    if (!a->kv[i] || (a->means && !kv_aligned(a->means[i], 16))) return VIREO_ERR_ARG;
    const gguf_kv_desc &x = a->kv[0]->d, &y = a->kv[i]->d;
    if (x.n_kv_heads != y.n_kv_heads || x.head_size != y.head_size || x.page_size != y.page_size ||
        x.n_pages != y.n_pages || x.kv_type != y.kv_type || x.page_stride != y.page_stride ||
        x.head_stride != y.head_stride || x.pos_stride != y.pos_stride)
      return VIREO_ERR_ARG;
  }
  if (a->n > 1 << 30) return VIREO_ERR_UNSUPPORTED;
  if (a->n == 0 || a->n_kv == 0) return VIREO_OK;
  int st;
  Ctx* c = ctx_get(&st);
  if (!c) return st;
  DeviceGuard dg(c->device);
  if (dg.status) return dg.status;
  const gguf_kv_desc& d = a->kv[0]->d;
  const int el = kv_type_size(d.kv_type);
  CopyParams p;
  p.src = a->src;
  p.dst = a->dst;
  p.rows = a->rows;
  p.n = a->n;
  p.n_pages = d.n_pages;
  p.page = d.page_size;
  p.G = d.n_kv_heads;
  p.chunk_shift = log2_of(d.head_size * el / 16);
  p.page_bytes = d.page_stride * el;
  p.head_bytes = d.head_stride * el;
  p.pos_bytes = d.pos_stride * el;
  p.heads_out = d.head_stride >= d.pos_stride;
  p.err = c->d_err;
  // whole pages, all pairs: 891 MB in 141.5 us instead of 144.5; a few pages are read again soon (a step's 10.5 MB:
  // 6.9 us through L2, 7.05 past it)
  p.stream = 2 * (int64_t)a->n_kv * a->n * d.n_kv_heads * d.page_size * d.head_size * el > (126ll << 20);
  // four chunks or more to a thread
  const int64_t units = (int64_t)d.n_kv_heads * d.page_size << p.chunk_shift;
  if (units > INT32_MAX / 2) return VIREO_ERR_UNSUPPORTED;
  p.group = 32;
  while (p.group < kCopyThreads && units > 4 * p.group) p.group *= 2;
  const int per = kCopyThreads / p.group;
  for (int l0 = 0; l0 < a->n_kv; l0 += kCopyLayers) {
    const int nl = std::min(kCopyLayers, a->n_kv - l0);
    for (int i = 0; i < nl; i++) {
      p.k[i] = (uint8_t*)a->kv[l0 + i]->d.k;
      p.v[i] = (uint8_t*)a->kv[l0 + i]->d.v;
      p.means[i] = a->means ? (uint8_t*)a->means[l0 + i] : nullptr;
    }
    if ((st = pdl_launch(kv_copy_kernel, dim3((unsigned)((a->n + per - 1) / per), 2 * nl), dim3(kCopyThreads), 0,
                         stream ? (cudaStream_t)stream : c->stream, p)))
      return st;
  }
  return VIREO_OK;
}

}  // extern "C"
