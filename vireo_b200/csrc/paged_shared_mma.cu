// Attention over prefixes that requests share, 16-bit caches: the units of
// paged_shared.cuh on the fifth-generation tensor cores.
//
// A unit is up to 128 rows (q heads of the requests that share the positions,
// or of one request) against a stretch of positions, in tiles.  Per tile
//
//   S = Q K^T      tcgen05.mma, rows x positions, fp32 in TMEM
//   P = 2^(S - m)  a thread per row; m the row's running maximum
//   O = P V        tcgen05.mma, P read from TMEM
//   acc = acc 2^(m_old - m) + O   in registers, to nearest
//
// O is taken out of TMEM tile by tile, so nothing in TMEM is ever rescaled and
// the tensor cores' own rounding of sums, towards zero, has one tile's length.
//
// P, and q where it is fp32, enter as two values of the cache's type, as in
// gguf_kv_attn: the upper one cut off, not rounded, so that both have one sign
// and an infinity times both stays itself.  P takes S's place in TMEM, 16
// positions (a step of the product) at a time: eight columns of upper
// values, eight of lower.
//
// Roles, in warpgroups: the softmax (row = thread; two of them take tiles in
// turn, each with a maximum and a sum of its own, so that neither waits for
// the other), the accumulators, and four warps: one issues the scores'
// products, one the values', so that neither waits for what the other waits
// for, and two load keys and values, each with a ring of its own.  The latter of
// these also brings a unit's q to shared memory once the last product with the
// one before is done.
//
// Neither limit is reached.  8 requests behind 131072 positions, 32 / 4 heads of 128,
// f32 / f16: this kernel 83 us cold (tensor pipe 52 %, HBM 41 %); with the join 82
// replayed, part of the 268 MB in L2, and 96 among other calls; floor 41.  64 behind
// 8192, bf16: 46 (24 %, 15 %), 46 and 47; floor 8.  The former is 5.8 thousand cycles a
// tile, the start included.  A further tile to every CTA adds 3.2 (bf16) to 4.1
// thousand while much comes from L2 and 5 or more where all comes from HBM, of which its
// products are 1.5 to 2.  What the rest goes to has not been shown: scores, maximum,
// weights, product and accumulators of a tile follow one another, with two tiles
// in work, one output in TMEM at 128 dimensions and two or three stages of keys and of
// values.  On CUDA cores the two cases took 883 and 1542 us; tiles of 64 positions at 128
// dimensions, with four buffers of scores, 58 and 125.  128 rows are the product's
// only shape for one CTA with a row to a thread; a unit of 8 rows, one request's
// own positions, costs the same per tile as one of 128.
#include <limits.h>

#include <type_traits>

#include "paged_shared.cuh"
#include "umma.cuh"

namespace vireo {

constexpr int kTcRows = 128;
constexpr int kTcMaxStages = 6;
constexpr int kTcSmem = 227 * 1024;

struct TcShared {
  uint64_t k_full[kTcMaxStages], k_empty[kTcMaxStages], v_full[kTcMaxStages], v_empty[kTcMaxStages];
  uint64_t images[2];          // of the first unit's rows written; of the others'
  uint64_t q_full[2], q_done[2];  // by unit: q there; every product with it done
  uint64_t s_full[3], p_full[3], s_empty[3];  // scores there; weights there; the product with them done
  uint64_t o_full[2], o_empty[2];
  uint64_t a_empty[2];            // maxima and sums read
  uint32_t tmem;
  int abort;
  float top[2][kTcRows], sum[2][kTcRows];  // by tile: the maximum its weights go by, the sum so far
};

template <class TA, int HS>
struct Tc {
  static constexpr bool kSplit = sizeof(TA) == 4;  // q as two values
  static constexpr int kTile = HS == 256 ? 64 : 128;
  static constexpr int kCols = HS / 64;                // 128-byte columns of a row
  static constexpr int kStage = kTile * HS * 2;        // bytes of a tile of keys or of values
  static constexpr int kQ = kTcRows * HS * 2;          // bytes of q, or of one of its two parts
  static constexpr int kQBytes = kSplit ? 2 * kQ : kQ;
  // By unit, the powers of two of q's rows.  With eight, those of unit u + 8 come
  // after the scores of unit u + 6, for which the softmax of the second tile of
  // unit u, at least, is done; with two stages of values or fewer, those of unit
  // u + 4 come after the values of unit u + 3, which says the same.
  static constexpr int kUps = !kSplit ? 0 : HS == 64 ? 8 : 4;
  static constexpr int kBudget = (kTcSmem - (int)sizeof(TcShared) - kUps * kTcRows - kQBytes) / kStage;
  static constexpr int kStages = kBudget < 2 * kTcMaxStages ? kBudget : 2 * kTcMaxStages;
  static constexpr int kK = (kStages + 1) / 2, kV = kStages / 2;
  // TMEM: scores of kS tiles, products of kO
  static constexpr int kS = 3, kO = HS == 64 ? 2 : 1;
  static constexpr int kSoft = HS == 256 ? 1 : 2;      // warpgroups of the softmax
  static constexpr int kAcc = HS == 64 ? 1 : 2;        // and of the accumulators,
  static constexpr int kDims = HS / kAcc;              // with so many dimensions each
  static constexpr int kThreads = 128 * (kSoft + kAcc + 1);
  // registers of a thread, at launch and then by role
  static constexpr int kRegs = 65536 / kThreads / 8 * 8;
  static constexpr int kRegSoft = HS == 64 ? 152 : 96, kRegAcc = HS == 64 ? 128 : HS == 128 ? 112 : 176,
                       kRegRest = HS == 64 ? 72 : 64;
  static_assert(kSoft * kRegSoft + kAcc * kRegAcc + kRegRest <= kRegs * kThreads / 128, "what the launch has");
  static constexpr int kImg = 1024 * kCols * (kSplit ? 2 : 1);  // eight rows of q
  static constexpr int kBytes = kQBytes + kStages * kStage + (int)sizeof(TcShared) + kUps * kTcRows;
  static_assert(kUps != 4 || kV <= 2, "as said");
  static_assert(kV >= 1 && kS * kTile + kO * HS <= 512 && kBytes <= kTcSmem, "fits an SM");
};
// Of q there is one tile in shared memory.  A unit of half as many rows or less
// takes the lower or the upper half in turn, in shared memory as in TMEM, so
// that the next one's are there before this one's last product.
constexpr int kTcHalf = kTcRows / 2;
VDEV int tc_place(int u, int rows) { return rows <= kTcHalf ? (u & 1) * kTcHalf : 0; }
template <int N>
VDEV void regs_more() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
VDEV void regs_less() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// D[tmem] (+)= A * B, A in shared memory or TMEM, B in shared memory; the warp
// executes it, so that its operands stay warp-wide values, and `lead` issues.
template <bool ACC>
VDEV void tc_mma_ss(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %5, 0;\n setp.ne.b32 q, %0, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%1], %2, %3, %4, p;\n}\n" ::"r"(lead),
      "r"(d), "l"(a), "l"(b), "r"(idesc), "n"(ACC ? 1 : 0));
}
template <bool ACC>
VDEV void tc_mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %5, 0;\n setp.ne.b32 q, %0, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%1], [%2], %3, %4, p;\n}\n" ::"r"(lead),
      "r"(d), "r"(a), "l"(b), "r"(idesc), "n"(ACC ? 1 : 0));
}
VDEV void tc_commit(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %0, 0;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n}\n" ::"r"(lead),
      "r"(smem_addr(bar))
      : "memory");
}
// Values: the product's columns are the dimensions, contiguous in a row of
// shared memory, so B is "MN-major": 64 dimensions to a 128-byte row, columns
// of such rows `col` bytes apart (leading offset), eight rows 1024 bytes apart
// (stride offset).
VDEV uint64_t umma_desc_mn(uint32_t addr, uint32_t col) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | (uint64_t)(col >> 4) << 16 | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
template <class TC>
__host__ __device__ constexpr uint32_t tc_idesc(int N, bool mn) {
  return umma_idesc_f16(kTcRows, N) | (std::is_same_v<TC, __nv_bfloat16> ? (1u << 7) | (1u << 10) : 0u) |
         (mn ? 1u << 16 : 0u);
}

#define TC_R16(v)                                                                                                  \
  "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]),       \
      "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
// 16 columns of the warp's lanes, on their way; they are there after tmem_ready
VDEV void tmem_ld16(uint32_t addr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(addr));
}
VDEV void tmem_ready(uint32_t (&v)[16]) { asm volatile("tcgen05.wait::ld.sync.aligned;" : TC_R16(v)::"memory"); }
VDEV void tmem_st16(uint32_t addr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
VDEV void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A warp's wait, with little code: the roles' loops share the instruction
// cache.  A try may take a microsecond; a wait that runs out of them (about 2 s)
// ends the call, everyone else's with it.
constexpr int kTcTries = 1 << 21;
VDEV bool tc_wait(TcShared* sh, uint64_t* bar, uint32_t parity, int* err) {
  for (int n = 0; n < kTcTries; n++) {
    if (mbar_test_suspend(bar, parity, 1000)) return true;
    if (*(volatile int*)&sh->abort) break;
  }
  *(volatile int*)&sh->abort = 1;
  set_error(err, VIREO_ERR_TIMEOUT);
  return false;
}
template <class T>
VDEV int8_t* tc_ups(TcShared* sh, int u) {
  return reinterpret_cast<int8_t*>(sh + 1) + u % T::kUps * kTcRows;
}
// a place in a ring of N: its t-th use
template <int N>
VDEV uint32_t tc_phase(int t) { return (uint32_t)(t / N) & 1u; }
// Waits for the arrivals of the last N of n uses: of commits each brings its own, in
// no order that is promised, and no product or arrival may be on its way when
// the CTA exits and its shared memory and TMEM are another's.  After a wait that
// ran out too, hence with its own limit and without a look at `abort`.
template <int N>
VDEV void tc_drain(uint64_t* bar, int n) {
  const int never = 0;
  for (int j = max(0, n - N); j < n; j++) mbar_wait_warp(&bar[j % N], tc_phase<N>(j), &never);
}

// ---- keys or values -----------------------------------------------------------
// before: what else the warp does for a unit, ahead of its tiles; false ends it
template <class T, int N, class F>
VDEV void tc_load(const ShParams& p, const CUtensorMap* map, const ShUnit* units, int nu, TcShared* sh, uint64_t* full,
                  uint64_t* empty, uint8_t* ring, F&& before) {
  constexpr int TILE = T::kTile;
  const int lane = threadIdx.x & 31, page = 1 << p.ps_shift, ppt = max(1, TILE >> p.ps_shift), rows = min(page, TILE);
  // page numbers are read a tile ahead: one read when its tile is due would
  // put its latency between any two tiles
  const auto page_of = [&](const ShUnit& x, int t) {
    const int i = (t * TILE >> p.ps_shift) + lane;
    return lane < ppt && i < (x.len + page - 1) >> p.ps_shift ? x.pages(p)[i] : 0;
  };
  int it = 0;
  ShUnit w = units[0], nx = units[min(1, nu - 1)];
  int pg = page_of(w, w.tile), last_rows = 0;
  bool ok = true;
#pragma unroll 1
  for (int u = 0; u < nu && ok; u++) {
    const ShUnit nn = units[min(u + 2, nu - 1)];
    const int next = page_of(nx, nx.tile);
    if (!(ok = before(w, u, last_rows))) break;
    last_rows = w.rows;
    const int end = w.tile + w.count, npages = (w.len + page - 1) >> p.ps_shift;
#pragma unroll 1
    for (int t = w.tile; t < end; t++, it++) {
      const int slot = it % N;
      const bool has = lane < ppt && (t * TILE >> p.ps_shift) + lane < npages;
      const int ahead = t + 1 < end ? page_of(w, t + 1) : next;
      const int cnt = __popc(__ballot_sync(0xffffffffu, has));
      if (it >= N) ok = __all_sync(0xffffffffu, tc_wait(sh, &empty[slot], tc_phase<N>(it) ^ 1u, p.err));
      if (!ok) break;
      if (lane == 0) mbar_arrive_expect_tx(&full[slot], (uint32_t)(cnt * rows * T::kCols * 128));
      __syncwarp();
      if (has) {
        if (pg < 0 || pg >= p.n_pages) {
          set_error(p.err, VIREO_ERR_ARG);
          pg = p.n_pages;  // outside the map: zeros
        }
        uint8_t* dst = ring + (size_t)slot * T::kStage + lane * rows * 128;
#pragma unroll
        for (int c = 0; c < T::kCols; c++)
          tma_load_4d(dst + c * TILE * 128, map, c * 64, (t * TILE) & (page - 1), w.kh, pg, &full[slot]);
      }
      pg = ahead;
    }
    w = nx;
    nx = nn;
  }
  tc_drain<N>(full, it);  // of copies too
}

// ---- products ----------------------------------------------------------------------
constexpr uint32_t kTcScores = 0;  // TMEM columns: of all of them the first is 0
// Scores, by a warp of their own.
template <class T, class TC, int HS>
VDEV void tc_scores(const ShParams& p, const ShUnit* units, int nu, TcShared* sh, uint32_t sq, uint32_t sk) {
  constexpr int TILE = T::kTile, KS = HS / 16;
  constexpr uint32_t qk = tc_idesc<TC>(TILE, false);
  constexpr uint64_t base = (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);  // as in umma_desc_sw128
  const uint32_t lead = (threadIdx.x & 31) == 0;
  const uint64_t q0 = base | (sq >> 4);
  int t = 0, u = 0;
  bool ok = true;
#pragma unroll 1
  for (; u < nu && ok; u++) {
    const int n = units[u].count;
#pragma unroll 1
    for (int i = 0; i < n && ok; i++, t++) {
      const int b = t % T::kS, slot = t % T::kK;
      ok = tc_wait(sh, &sh->k_full[slot], tc_phase<T::kK>(t), p.err);
      if (i == 0) ok = ok && tc_wait(sh, &sh->q_full[u & 1], tc_phase<2>(u), p.err);
      if (t >= T::kS) ok = ok && tc_wait(sh, &sh->s_empty[b], tc_phase<T::kS>(t) ^ 1u, p.err);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      tc_fence_after();
      const uint32_t d = kTcScores + b * TILE;
      const uint64_t k0 = base | ((sk + slot * T::kStage) >> 4);
      // Lower values first: sums are cut towards zero at every step, the small
      // ones where that costs little (8 requests behind 131072 positions, f32: the
      // output off by 1.4e-6 with lower values last, and between the weights' upper
      // ones).
#pragma unroll
      for (int part = T::kSplit ? 1 : 0; part >= 0; part--)
#pragma unroll
        for (int k = 0; k < KS; k++) {
          const uint64_t qd = q0 + (part * T::kQ + (k >> 2) * kTcRows * 128 + (k & 3) * 32) / 16,
                         kd = k0 + ((k >> 2) * TILE * 128 + (k & 3) * 32) / 16;
          if (part == (T::kSplit ? 1 : 0) && k == 0)
            tc_mma_ss<false>(lead, d, qd, kd, qk);
          else
            tc_mma_ss<true>(lead, d, qd, kd, qk);
        }
      tc_commit(lead, &sh->s_full[b]);
      tc_commit(lead, &sh->k_empty[slot]);
      if (i == n - 1) tc_commit(lead, &sh->q_done[u & 1]);
    }
  }
  tc_drain<T::kS>(sh->s_full, t);
  tc_drain<T::kK>(sh->k_empty, t);
  tc_drain<2>(sh->q_done, ok ? u : u - 1);
}
// Weights times values, by another.
template <class T, class TC, int HS>
VDEV void tc_values(const ShParams& p, const ShUnit* units, int nu, TcShared* sh, uint32_t sv) {
  constexpr int TILE = T::kTile;
  constexpr uint32_t pv = tc_idesc<TC>(HS, true);
  const uint32_t lead = (threadIdx.x & 31) == 0;
  int t = 0;
  bool ok = true;
#pragma unroll 1
  for (int u = 0; u < nu && ok; u++) {
    const int n = units[u].count, behind = units[u].len - units[u].tile * TILE;
#pragma unroll 1
    for (int i = 0; i < n && ok; i++, t++) {
      const int b = t % T::kS, o = t % T::kO, slot = t % T::kV, valid = behind - i * TILE;
      ok = tc_wait(sh, &sh->v_full[slot], tc_phase<T::kV>(t), p.err);
      if (valid % 16 && valid < TILE) {
        // value rows behind the last position that the product takes in: zeros,
        // since their weight of zero does not cancel a NaN
        const uint32_t at = sv + slot * T::kStage + valid * 128, more = (16 - valid % 16) * 128;
        for (int c = 0; c < T::kCols; c++)
          for (uint32_t x = 16 * (threadIdx.x & 31); x < more; x += 512)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at + c * TILE * 128 + x), "r"(0) : "memory");
        fence_proxy_async();
        __syncwarp();
      }
      ok = ok && tc_wait(sh, &sh->p_full[b], tc_phase<T::kS>(t), p.err);
      if (t >= T::kO) ok = ok && tc_wait(sh, &sh->o_empty[o], tc_phase<T::kO>(t) ^ 1u, p.err);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      tc_fence_after();
      const uint32_t a = kTcScores + b * TILE, d = kTcScores + T::kS * TILE + o * HS;
      const uint64_t v = umma_desc_mn(sv + slot * T::kStage, TILE * 128);
      const int steps = min(TILE, valid + 15) / 16;  // with positions
      tc_mma_ts<false>(lead, d, a + 8, v, pv);  // lower values first, as above
#pragma unroll
      for (int k = 1; k < TILE / 16; k++)
        if (k < steps) tc_mma_ts<true>(lead, d, a + 16 * k + 8, v + k * 128, pv);
#pragma unroll
      for (int k = 0; k < TILE / 16; k++)
        if (k < steps) tc_mma_ts<true>(lead, d, a + 16 * k, v + k * 128, pv);
      tc_commit(lead, &sh->o_full[o]);
      tc_commit(lead, &sh->s_empty[b]);
      tc_commit(lead, &sh->v_empty[slot]);
    }
  }
  tc_drain<T::kO>(sh->o_full, t);
  tc_drain<T::kS>(sh->s_empty, t);
  tc_drain<T::kV>(sh->v_empty, t);
}

// 2^e of a normal result
VDEV float tc_pow2(int e) { return __int_as_float((e + 127) << 23); }

// Two values as f16, cut off, and what that leaves, rounded: of one sign, and no
// zero beside a value (an infinite key times it would be no number).  An
// infinity leaves the least there is.
VDEV void tc_split(float a, float b, uint32_t& hi, uint32_t& lo) {
  asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(b), "f"(a));
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  lo = pack_h2(a - h.x, b - h.y);
  const uint32_t none = __vcmpeq2(lo & 0x7fff7fffu, 0u) & ~__vcmpeq2(hi & 0x7fff7fffu, 0u);
  const uint32_t top = __vcmpeq2(hi & 0x7fff7fffu, 0x7c007c00u);
  lo = (lo & ~(none | top)) | ((none | top) & ((hi & 0x80008000u) | 0x00010001u));
}

// ---- q -----------------------------------------------------------------------------
// Every unit's rows as the products read them, to global memory first: eight
// rows of 128 bytes lie together, 16-byte chunk c of row r at (c ^ r) & 7; behind
// them the other dimensions, 64 at a time, and the lower values of fp32 rows.
// Those are scaled by a power of two, kept in p.up; the scale's sign goes into q.
// One warp's conversion of a unit's rows, when they were due, took as long as
// three tiles.  first .. last: eights of the CTA's, by warps `warp` of NW.
template <class T, class TA, int HS, int NW>
VDEV void tc_images(const ShParams& p, const ShStretch& my, int first, int last, int warp) {
  constexpr int E = 16 / (int)sizeof(TA), LPR = HS / E, CPL = LPR > 32 ? LPR / 32 : 1, RPI = LPR < 32 ? 32 / LPR : 1;
  constexpr int STEPS = 8 / RPI, U = CPL > 1 ? 2 : 4;  // of eight rows; taken together
  const int lane = threadIdx.x & 31, sub = lane / LPR, c0 = LPR < 32 ? lane % LPR : lane;
  const auto rows_of = [&](int s) { return p.eights[my.img + min(s, last * STEPS - 1) / STEPS]; };
  ShEight w[U], ahead[U];
#pragma unroll
  for (int j = 0; j < U; j++) ahead[j] = rows_of(first * STEPS + warp + j * NW);
#pragma unroll 1
  for (int s0 = first * STEPS + warp; s0 < last * STEPS; s0 += U * NW) {
    uint4 x[U][CPL];
    int r[U];
    bool has[U];
#pragma unroll
    for (int j = 0; j < U; j++) {
      w[j] = ahead[j];
      ahead[j] = rows_of(s0 + (U + j) * NW);
    }
#pragma unroll
    for (int j = 0; j < U; j++) {
      const int s = s0 + j * NW, n = s < last * STEPS ? w[j].n_kh & 15 : 0;
      r[j] = s % STEPS * RPI + sub;
      has[j] = r[j] < n;
#pragma unroll
      for (int c = 0; c < CPL; c++) x[j][c] = make_uint4(0u, 0u, 0u, 0u);
      if (has[j]) {
        const int f = w[j].row + r[j], m = f / p.R;
        const TA* q = reinterpret_cast<const TA*>(p.q) + (int64_t)(w[j].seq + m) * p.q_stride +
                      (int64_t)((w[j].n_kh >> 4) * p.R + f - m * p.R) * HS;
#pragma unroll
        for (int c = 0; c < CPL; c++) x[j][c] = *(reinterpret_cast<const uint4*>(q) + c0 + 32 * c);
      }
    }
    float mx[U];
    if constexpr (T::kSplit) {
#pragma unroll
      for (int j = 0; j < U; j++) {
        mx[j] = 0.f;
#pragma unroll
        for (int c = 0; c < CPL; c++) {
          const float4 v = *reinterpret_cast<const float4*>(&x[j][c]);
          mx[j] = fmaxf(fmaxf(fmaxf(mx[j], fabsf(v.x)), fmaxf(fabsf(v.y), fabsf(v.z))), fabsf(v.w));
        }
      }
#pragma unroll
      for (int o = (LPR < 32 ? LPR : 32) / 2; o; o >>= 1)
#pragma unroll
        for (int j = 0; j < U; j++) mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], o));
    }
#pragma unroll
    for (int j = 0; j < U; j++) {
      const int at = my.img + (s0 + j * NW) / STEPS;
      uint8_t* to = p.img + (int64_t)at * T::kImg + r[j] * 128;
      if constexpr (T::kSplit) {
        // the largest to [2^14, 2^15), as in gguf_kv_attn
        const int e = mx[j] > 0.f ? min(max((__float_as_int(mx[j]) >> 23) - 127, -112), 127) - 14 : 0;
        const float down = p.scale < 0.f ? -tc_pow2(-e) : tc_pow2(-e);
        if (has[j] && c0 == 0) p.up[(int64_t)at * 8 + r[j]] = (int8_t)e;
#pragma unroll
        for (int c = 0; c < CPL; c++) {
          const float4 v4 = *reinterpret_cast<const float4*>(&x[j][c]);
          uint2 hi, lo;
          tc_split(v4.x * down, v4.y * down, hi.x, lo.x);
          tc_split(v4.z * down, v4.w * down, hi.y, lo.y);
          const int ch = 4 * (c0 + 32 * c);  // first dimension
          uint8_t* d = to + (ch >> 6) * 1024 + (((ch >> 3 & 7) ^ (r[j] & 7)) << 4) + (ch & 4) * 2;
          if (has[j]) {
            *reinterpret_cast<uint2*>(d) = hi;
            *reinterpret_cast<uint2*>(d + T::kCols * 1024) = lo;
          }
        }
      } else {
        uint4 v = x[j][0];
        if (p.scale < 0.f) {
          v.x ^= 0x80008000u;
          v.y ^= 0x80008000u;
          v.z ^= 0x80008000u;
          v.w ^= 0x80008000u;
        }
        if (has[j]) *reinterpret_cast<uint4*>(to + (c0 >> 3) * 1024 + (((c0 & 7) ^ (r[j] & 7)) << 4)) = v;
      }
    }
  }
  asm volatile("fence.proxy.async;" ::: "memory");  // copies read them
}
// A unit's image to shared memory, once every product with what lies there is
// done: the last unit's, or the one's before where both take halves.  The first
// unit's images come from all of softmax and accumulators, the others' from the
// latter, who have time until the first weights are there.  Whoever has written
// arrives and goes on; this warp alone waits.
template <class T>
VDEV bool tc_bring(const ShParams& p, const ShUnit& w, int u, int last_rows, TcShared* sh, uint8_t* sq) {
  bool ok = u >= 2 || tc_wait(sh, &sh->images[u], 0, p.err);
  constexpr int N = T::kCols * (T::kSplit ? 2 : 1);
  const int lane = threadIdx.x & 31, eights = (w.rows + 7) / 8, place = tc_place(u, w.rows);
  uint32_t ups = 0;
  if (T::kSplit && lane < 2 * eights)
    ups = *reinterpret_cast<const uint32_t*>(p.up + (int64_t)w.img * 8 + 4 * lane);
  const int v = w.rows > kTcHalf || last_rows > kTcHalf ? u - 1 : u - 2;
  ok = ok && (v < 0 || tc_wait(sh, &sh->q_done[v & 1], tc_phase<2>(v), p.err));
  if (!__all_sync(0xffffffffu, ok)) return false;
  if constexpr (T::kSplit)
    if (lane < 2 * eights) *reinterpret_cast<uint32_t*>(tc_ups<T>(sh, u) + place + 4 * lane) = ups;
  __syncwarp();
  if (lane == 0) mbar_arrive_expect_tx(&sh->q_full[u & 1], (uint32_t)(eights * N * 1024));
  __syncwarp();
  for (int i = lane; i < eights * N; i += 32) {
    const int e = i / N, j = i % N;
    bulk_g2s(sq + j / T::kCols * T::kQ + j % T::kCols * kTcRows * 128 + (place / 8 + e) * 1024,
             p.img + (int64_t)(w.img + e) * T::kImg + j * 1024, 1024, &sh->q_full[u & 1]);
  }
  __syncwarp();
  return true;
}

// ---- softmax, a thread per row ---------------------------------------------------
template <class T, class TC, int HS>
VDEV void tc_softmax(const ShParams& p, const ShUnit* units, int nu, TcShared* sh) {
  constexpr int TILE = T::kTile;
  constexpr bool F16 = std::is_same_v<TC, __half>;
  const int row = threadIdx.x & 127, warp = row >> 5, me = (int)threadIdx.x >> 7;
  const uint32_t lanes = (uint32_t)(32 * warp) << 16;
  int t = 0;
#pragma unroll 1
  for (int u = 0; u < nu; u++) {
    const int n = units[u].count, behind = units[u].len - units[u].tile * TILE, place = tc_place(u, units[u].rows);
    const bool busy = 32 * warp + 31 >= place && 32 * warp < place + units[u].rows;
    float qs = 0.f;
    float raw = -INFINITY, m = -INFINITY, l = 0.f;  // the largest score as the product has it, and scaled
#pragma unroll 1
    for (int i = 0; i < n; i++, t++) {
      if (T::kSoft > 1 && t % T::kSoft != me) continue;
      const int b = t % T::kS, valid = behind - i * TILE;  // positions of this tile, or more
      const uint32_t s_at = sh->tmem + lanes + b * TILE;
      tc_wait(sh, &sh->s_full[b], tc_phase<T::kS>(t), p.err);
      tc_fence_after();
      if (busy) {
        if (qs == 0.f) {  // the unit's first of this warpgroup
          qs = fabsf(p.scale);
          if constexpr (T::kSplit) qs *= tc_pow2(tc_ups<T>(sh, u)[row]);
          qs = fmaxf(qs, 1.40129846e-45f);  // the least there is: a score of -inf stays one
        }
        // 16 columns (a step of the values' product) at a time, the next ones on
        // their way; columns behind the last position as scores of -inf.  The
        // loops stay rolled: unrolled over a tile, with the other roles' code
        // between, they waited for instructions more than for anything else.
        uint32_t xa[16], xb[16];
        const auto cut = [&](int c, uint32_t(&s)[16]) {
          if (c + 16 > valid)
#pragma unroll
            for (int j = 0; j < 16; j++) s[j] = c + j < valid ? s[j] : 0xff800000u;
        };
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        const auto most = [&](int c, uint32_t(&s)[16]) {
          cut(c, s);
#pragma unroll
          for (int j = 0; j < 16; j++) mx[j & 3] = fmaxf(mx[j & 3], __uint_as_float(s[j]));
        };
        tmem_ld16(s_at, xa);
        const int cols = min(TILE, valid);
#pragma unroll 1
        for (int c = 0; c < cols; c += 32) {
          tmem_ready(xa);
          tmem_ld16(s_at + c + 16, xb);
          most(c, xa);
          tmem_ready(xb);
          tmem_ld16(s_at + (c + 32 < cols ? c + 32 : 0), xa);  // behind the last, the first again
          most(c + 16, xb);
        }
        raw = fmaxf(raw, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
        const float mn = __fmul_rn(raw, qs), sub = raw == -INFINITY ? 0.f : mn;  // scores of -inf alone
        l *= sh_ex2(m - sub);
        m = mn;
        // What the maximum lost in its rounding: the scores' products lose nothing where it is
        // taken off, so all weights would have that too much or too little in their power,
        // which of maxima from 2^25 on is more than f16 holds, and of larger ones than anything.
        const float lost = raw == -INFINITY ? 0.f : fmaf(raw, qs, -mn);
        // weights up to 2^14 over f16, as in gguf_kv_attn
        const float up = (F16 ? 14.f : 0.f) - lost;
        const f2 qq = f2_make(qs, qs), mm = f2_make(-sub, -sub), rest = f2_make(up, up);
        f2 sums[2] = {f2_make(0.f, 0.f), f2_make(0.f, 0.f)};
        const auto weigh = [&](int c, uint32_t(&s)[16]) {
          cut(c, s);
          uint32_t y[16];  // eight columns of upper values, eight of lower
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            f2 d = f2_fma(f2_make(__uint_as_float(s[j]), __uint_as_float(s[j + 1])), qq, mm);
            d = f2_add(d, rest);
            float d0, d1;
            f2_get(d, d0, d1);
            const float e0 = sh_ex2(d0), e1 = sh_ex2(d1);
            sums[j / 2 & 1] = f2_add(sums[j / 2 & 1], f2_make(e0, e1));
            constexpr uint32_t keep = F16 ? 0xffffe000u : 0xffff0000u;
            const float h0 = __uint_as_float(__float_as_uint(e0) & keep), h1 = __uint_as_float(__float_as_uint(e1) & keep);
            if constexpr (F16) {
              y[j / 2] = pack_h2(h0, h1);
              y[j / 2 + 8] = pack_h2(e0 - h0, e1 - h1);
            } else {
              y[j / 2] = __byte_perm(__float_as_uint(e0), __float_as_uint(e1), 0x7632);
              const __nv_bfloat162 lo = __floats2bfloat162_rn(e0 - h0, e1 - h1);
              y[j / 2 + 8] = *reinterpret_cast<const uint32_t*>(&lo);
            }
          }
          tmem_st16(s_at + c, y);
        };
#pragma unroll 1
        for (int c = 0; c < cols; c += 32) {
          tmem_ready(xa);
          tmem_ld16(s_at + c + 16, xb);
          weigh(c, xa);
          tmem_ready(xb);
          tmem_ld16(s_at + (c + 32 < cols ? c + 32 : 0), xa);  // behind the last, what nobody looks at
          weigh(c + 16, xb);
        }
        tmem_ready(xa);
        float a0, a1;
        f2_get(f2_add(sums[0], sums[1]), a0, a1);
        l += a0 + a1;
        tmem_st_wait();
      }
      if (t >= 2) tc_wait(sh, &sh->a_empty[t & 1], tc_phase<2>(t) ^ 1u, p.err);
      sh->top[t & 1][row] = m;
      sh->sum[t & 1][row] = l;
      tc_fence_before();
      mbar_arrive(&sh->p_full[b]);
    }
  }
}

// ---- accumulators: rows of a warpgroup's dimensions ---------------------------------
template <class T, int HS>
VDEV void tc_accumulate(const ShParams& p, const ShUnit* units, int nu, TcShared* sh) {
  constexpr int D = T::kDims;
  const int g = ((int)threadIdx.x >> 7) - T::kSoft, row = threadIdx.x & 127, warp = row >> 5;
  const uint32_t o_at = kTcScores + T::kS * T::kTile + D * g + ((uint32_t)(32 * warp) << 16);
  int t = 0;
#pragma unroll 1
  for (int u = 0; u < nu; u++) {
    const int n = units[u].count, nr = units[u].rows, place = tc_place(u, nr);
    const bool busy = 32 * warp + 31 >= place && 32 * warp < place + nr;
    f2 acc[D / 2];
#pragma unroll
    for (int j = 0; j < D / 2; j++) acc[j] = f2_make(0.f, 0.f);
    float M = -INFINITY, m0 = -INFINITY, l0 = 0.f, m1 = -INFINITY, l1 = 0.f;  // of the last two tiles
#pragma unroll 1
    for (int i = 0; i < n; i++, t++) {
      const int o = t % T::kO;
      tc_wait(sh, &sh->o_full[o], tc_phase<T::kO>(t), p.err);
      tc_wait(sh, &sh->p_full[t % T::kS], tc_phase<T::kS>(t), p.err);
      tc_fence_after();
      if (T::kSoft > 1) {
        m1 = m0;
        l1 = l0;
      }
      m0 = sh->top[t & 1][row];
      l0 = sh->sum[t & 1][row];
      mbar_arrive(&sh->a_empty[t & 1]);
      if (busy) {
        const float mn = fmaxf(M, m0), sub = mn == -INFINITY ? 0.f : mn;
        const float a = sh_ex2(M - sub), f = sh_ex2(m0 - sub);
        M = mn;
        const f2 aa = f2_make(a, a), ff = f2_make(f, f);
        uint32_t x[2][16];
        tmem_ld16(o_at + o * HS, x[0]);
#pragma unroll
        for (int c = 0; c < D; c += 16) {
          uint32_t(&y)[16] = x[c / 16 & 1];
          tmem_ready(y);
          if (c + 16 < D) {
            tmem_ld16(o_at + o * HS + c + 16, x[(c / 16 & 1) ^ 1]);
          } else {  // all read: the next product may come
            tc_fence_before();
            mbar_arrive(&sh->o_empty[o]);
          }
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            f2& v = acc[(c + j) / 2];
            v = f2_fma(v, aa, f2_mul(f2_make(__uint_as_float(y[j]), __uint_as_float(y[j + 1])), ff));
          }
        }
      } else {
        mbar_arrive(&sh->o_empty[o]);
      }
    }
    if (row >= place && row < place + nr) {
      const float sub = M == -INFINITY ? 0.f : M;
      float* part = p.part + (int64_t)(units[u].part + row - place) * (HS + 4);
#pragma unroll
      for (int j = 0; j < D / 4; j++) {
        float v[4];
        f2_get(acc[2 * j], v[0], v[1]);
        f2_get(acc[2 * j + 1], v[2], v[3]);
        store_f<4>(part + D * g + 4 * j, v);
      }
      if (g == 0) {
        part[HS] = M;
        part[HS + 1] = l0 * sh_ex2(m0 - sub) + l1 * sh_ex2(m1 - sub);
      }
    }
  }
}

template <class TA, class TC, int HS>
__global__ void __launch_bounds__(Tc<TA, HS>::kThreads, 1)
    sh_mma(const __grid_constant__ ShParams p, const __grid_constant__ CUtensorMap map_k,
           const __grid_constant__ CUtensorMap map_v) {
  using T = Tc<TA, HS>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t *sq = smem, *sk = sq + T::kQBytes, *sv = sk + T::kK * T::kStage;
  TcShared* sh = reinterpret_cast<TcShared*>(sv + T::kV * T::kStage);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kTcMaxStages; i++) {
      mbar_init(&sh->k_full[i], 1);
      mbar_init(&sh->k_empty[i], 1);
      mbar_init(&sh->v_full[i], 1);
      mbar_init(&sh->v_empty[i], 1);
    }
    mbar_init(&sh->images[0], 128 * (T::kSoft + T::kAcc));
    mbar_init(&sh->images[1], 128 * T::kAcc);
    for (int i = 0; i < 3; i++) {
      mbar_init(&sh->s_full[i], 1);
      mbar_init(&sh->p_full[i], kTcRows);
      mbar_init(&sh->s_empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&sh->q_full[i], 1);
      mbar_init(&sh->q_done[i], 1);
      mbar_init(&sh->o_full[i], 1);
      mbar_init(&sh->o_empty[i], 128 * T::kAcc);
      mbar_init(&sh->a_empty[i], 128 * T::kAcc);
    }
    sh->abort = 0;
    mbar_fence_init();
  }
  if (warp == 0) tmem_alloc(&sh->tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();  // whoever comes next finds TMEM taken and does not keep it from this CTA
  pdl_wait();
  const ShStretch my = sh_plan<T::kThreads, true>(p, smem);
  const ShUnit* units = my.units;
  const int nu = my.n;
  constexpr int first = 4 * (T::kSoft + T::kAcc);
  if (warp < first && nu > 0) {
    tc_images<T, TA, HS, first>(p, my, 0, (units[0].rows + 7) / 8, warp);
    mbar_arrive(&sh->images[0]);
  }
  if (warp < 4 * T::kSoft) {
    if constexpr (T::kRegSoft > T::kRegs) regs_more<T::kRegSoft>();
    if constexpr (T::kRegSoft < T::kRegs) regs_less<T::kRegSoft>();
    tc_softmax<T, TC, HS>(p, units, nu, sh);
  } else if (warp < first) {
    if constexpr (T::kRegAcc > T::kRegs) regs_more<T::kRegAcc>();
    if (nu > 1) {
      tc_images<T, TA, HS, 4 * T::kAcc>(p, my, (units[0].rows + 7) / 8, my.eights, warp - 4 * T::kSoft);
      mbar_arrive(&sh->images[1]);
    }
    tc_accumulate<T, HS>(p, units, nu, sh);
  } else {
    regs_less<T::kRegRest>();
    if (nu > 0) {
      if (warp == first)
        tc_scores<T, TC, HS>(p, units, nu, sh, smem_addr(sq), smem_addr(sk));
      else if (warp == first + 1)
        tc_values<T, TC, HS>(p, units, nu, sh, smem_addr(sv));
      else if (warp == first + 2)
        tc_load<T, T::kK>(p, &map_k, units, nu, sh, sh->k_full, sh->k_empty, sk, [](const ShUnit&, int, int) { return true; });
      else {
        int brought = 0;
        tc_load<T, T::kV>(p, &map_v, units, nu, sh, sh->v_full, sh->v_empty, sv, [&](const ShUnit& w, int u, int last) {
          const bool ok = tc_bring<T>(p, w, u, last, sh, sq);
          brought += ok;
          return ok;
        });
        tc_drain<2>(sh->q_full, brought);
      }
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(sh->tmem, 512);
}

template <class TA, class TC, int HS>
static ShKernel tc_kernel() {
  using T = Tc<TA, HS>;
  return {reinterpret_cast<const void*>(&sh_mma<TA, TC, HS>), T::kThreads, T::kBytes, kTcRows, T::kTile, true, T::kImg,
          1};
}
template <class TA, class TC>
static ShKernel tc_kernel_h(int hs) {
  return hs == 64 ? tc_kernel<TA, TC, 64>() : hs == 128 ? tc_kernel<TA, TC, 128>() : tc_kernel<TA, TC, 256>();
}
ShKernel sh_mma_kernel(const gguf_kv_desc& d) {
  if (d.act_type == KV_BF16) return tc_kernel_h<__nv_bfloat16, __nv_bfloat16>(d.head_size);
  return d.act_type == KV_F16 ? tc_kernel_h<__half, __half>(d.head_size) : tc_kernel_h<float, __half>(d.head_size);
}

}  // namespace vireo
