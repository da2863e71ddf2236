// Attention of drafted tokens that form a tree over the paged shared-KV caches (sm_100a).
//
// A request's n drafted tokens sit in the window cache at slots [ctx, ctx + n)
// (ctx = seqused_kv - n); parents[i] < i is the token that i follows, -1 the
// cached context, anything below an unused slot. Token i at depth d has
// position s = ctx + d and attends to
//   the cached rows [s - win, ctx), its ancestors no more than win back, itself;
//   compressed rows below ctx // ratio: all of them, or its top-k list.
// o = sum_j p_j v_j / (sum_j p_j + e^sink),  p_j = e^(scale q.k_j),  K = V.
//
// Work: one unit is 128 (token, head) rows of one request, in order, so a
// request's units read the same rows; with top-k lists a unit is 128 heads of
// one token. A unit's rows of KV come in tiles of 128: the window (cached and
// drafted rows together), then the compressed ones. All tiles of all units
// form one sequence that is cut into equal ranges, one per pair of CTAs; a unit
// cut by a range's end leaves partial sums that tree_combine_kernel joins in order.
//
// A pair of CTAs (one cluster) works on a unit, 64 rows each, with tcgen05.mma
// over both SMs (cta_group::2, M = 128): S[128 x 128] = Q K^T, each CTA
// bringing 64 of the tile's rows as K, and O[128 x 512] += P V, each bringing
// 256 of the 512 columns as V. Why: O of 128 rows fills the tensor memory of
// one SM, of 64 rows half of it, but one SM's M = 64 runs at half rate (64
// cycles for N = 128; 48 in the weight-stationary form), where the pair runs at
// 45.6 (N = 128) and the full rate of 64 (N = 256), all measured; and K and V,
// 64 KB each, are then separate buffers, so that the next tile's K is copied
// and multiplied while this tile's softmax runs. The accumulators use all 128
// TMEM lanes (lanes 64-127 hold the upper half of the columns): two buffers of S
// take 64 columns each, O two of three places of 128, in turn: half q of the
// sequence of the units' halves has place q % 3, so that a unit's products begin
// while the unit before it is read.
// The softmax is one pass with a running maximum that moves, and rescales O,
// only when a row's maximum rises by more than 2^8: P then stays below 2^8, and
// P, l and O keep one common scale. P is rounded to the I/O type for the product,
// whose operands have one type; l sums it unrounded (both as the framework's
// forward does). It is the one rounding before the result's, and takes the result
// from 1.7e-3 to 2.1e-3 off the 64-bit one in bf16, 2.1e-4 to 2.6e-4 in fp16 (norms).
//
// Roles (23 warps), each of which walks the ring of published tiles by itself:
//   0-7    softmax: thread = row, 32 of the tile's columns;
//   8-11   epilogue: O of a finished unit leaves while the next one runs;
//   12, 13 issue the scores and the products (first CTA), or tell the first CTA
//          that this one's K and Q, or V, have landed (second CTA);
//   14     coordinator: walks the range and the trees, works out which rows each
//          token sees and publishes tiles (the pair's two take the same steps);
//   15-18  copy Q and K, 19-22 V.
// What bounds it. The products of a tile take 2500 cycles. With about 20 us that a call
// of any size takes (a single tile through every role and the joining kernel, 21 us)
// left out, a tile takes 4800 over the whole cache (16 trees of 32 tokens x 128 heads
// over 65k-262k: 59 tiles a pair, 165 us at 1965 MHz, 762 TFLOP/s, 46% of the
// library's bf16 rate; tensor pipe 42% busy): the softmax warps' serial chain per
// tile, some 400 instructions and 12 round trips to shared memory and barriers
// between the scores and P. With lists it takes 6400 (64 x 8 x 128 heads, 512 of
// them: 32 tiles a pair, 125 us, 2.1 TB/s, DRAM 31% busy): the same chain, and copies
// by cp.async in the place of boxes; how much of the difference is theirs was not
// measured by itself. Window alone (127, 64 trees of 16 x 64 heads: two tiles a unit,
// the second nearly empty, 70 us): ends of units. Neither memory nor L2 (30%) is near
// its rate. A chain of drafted tokens costs the coordinator a walk up it for every
// unit: 8 chains of 1024 x 8 heads take 770 us, where their tiles are worth some 200.
// Measured and left out: registers moved between warps (setmaxnreg, slower), P
// before the row's maximum is known and again if it moved (3% slower), output rows
// stored from registers (slower).
// Copies: Q, and the rows of pages of a multiple of 64, are TMA boxes of 64 rows
// x 64 columns issued by one thread (window tiles then begin at a multiple of 64,
// so that 64 rows never leave a page). Top-k rows and other pages take cp.async,
// one row's 512 bytes per instruction, whose 256 instructions a tile hold up
// every other warp's shared-memory accesses.
#include <cuda.h>

#include <mutex>

#include "sas_common.cuh"

namespace {

constexpr int D = 512;
constexpr int MR = 64;    // rows of a CTA
constexpr int UR = 128;   // rows of a unit
constexpr int CH = 128;   // KV rows of a tile
constexpr int kMaxTok = 8;      // tokens of a CTA's rows: heads are a multiple of 8
constexpr int kMaxUnitTok = 16;
constexpr int kMaxTree = 1024;  // drafted tokens of a request
constexpr int kWords = kMaxTree / 32;
constexpr int kMaxCtx = 1 << 30;  // rows cached before them
constexpr int KSLAB = 64 * 128;   // 64 columns of the CTA's 64 K rows
constexpr int VSLAB = CH * 128;   // 64 columns of the tile's V rows
constexpr int QSLAB = MR * 128;   // 64 columns of Q, or of P
constexpr int kSmWarps = 8, kEpiWarp0 = 8, kEpiWarps = 4, kQkWarp = 12, kPvWarp = 13, kCoordWarp = 14, kKWarp0 = 15, kVWarp0 = 19,
              kLoadWarps = 4;
constexpr int kThreads = 32 * 23;
constexpr int kRing = 7;          // tiles the coordinator may be ahead (5: up to 1% slower)
constexpr int kUnitSlots = 9;     // > kRing + 1: no slot is rewritten while a published tile names it
constexpr uint32_t TM_O = 0, TM_S = 384, TM_COLS = 512;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kMove = 8.f;      // log2 units the running maximum may lag

constexpr int OFF_Q = 0;
constexpr int OFF_K = OFF_Q + 8 * QSLAB;
constexpr int OFF_V = OFF_K + 8 * KSLAB;
constexpr int OFF_P = OFF_V + 4 * VSLAB;
constexpr int OFF_MISC = OFF_P + 2 * QSLAB;

// X* count in the first CTA: the second's copies have landed. So do SEMPTY (the
// scores are read), PREADY and OEMPTY, on which both CTAs' warps arrive.
// K and V come in two halves of their columns, each with its own barriers, so
// that the next tile's first half is on its way while the second is multiplied.
enum Bar { B_KFULL = 0, B_VFULL = 2, B_QFULL = 4, B_XK, B_XV = B_XK + 2, B_XQ = B_XV + 2, B_KEMPTY, B_VEMPTY = B_KEMPTY + 2,
           B_QEMPTY = B_VEMPTY + 2, B_MASK, B_SFULL = B_MASK + 3, B_SEMPTY = B_SFULL + 2, B_PREADY = B_SEMPTY + 2, B_OFULL, B_OEMPTY,
           B_FIN = B_OEMPTY + 3, B_SSYNC = B_FIN + 2, B_CFULL = B_SSYNC + 2, B_CEMPTY = B_CFULL + kRing, B_DRAIN = B_CEMPTY + kRing, B_COUNT = B_DRAIN + 2 };

// Waits, as the status word names them: SAS_ERR_TIMEOUT_BASE + id, those of the forward
// below 20. One for each place that waits; both halves and both buffers of a thing share it.
enum WaitId : int {
  W_UNIT_SLOT = 20, W_PUBLISH, W_LOAD_TILE, W_Q_FREE, W_K_FREE, W_V_FREE,         // coordinator, loaders
  W_MMA_TILE, W_PASS_Q, W_PASS_K, W_PASS_V,                                       // issuers, second CTA
  W_PV_P, W_PV_O, W_PV_V, W_PV_XV, W_QK_Q, W_QK_XQ, W_QK_S, W_QK_K, W_QK_XK,      // issuers, first CTA
  W_EPI_UNIT, W_EPI_O,                                                            // epilogue
  W_SM_TILE, W_SM_END, W_SM_MASK, W_SM_S, W_SM_V_FREE, W_SM_V, W_SM_MAX, W_SM_P   // softmax
};

enum TileFlag : int {
  TF_FIRST = 1, TF_LAST = 2, TF_END = 4, TF_ZERO = 8,  // ZERO: no token of the unit is in use, its output is zero
  TF_CMP = 16, TF_TOPK = 32, TF_PART0 = 64, TF_PART1 = 128  // PARTn: the piece goes to the CTA's partial n
};

struct Tile { int flags, row0, nrows, uslot; };
struct Unit {
  int b, tok, ctx, thr;      // tok: first token
  int64_t qrow;              // first row of [T * H]
  int nrows, roff;           // roff: head of the first row
  int pos[kMaxTok];          // s of each token, -1: unused
};
struct Fin {  // a finished unit, from the softmax warps to the epilogue
  float m[MR], l[4][MR];     // l: of a quarter of the columns; < 0 in the first: the row's token is not in use
  int64_t qrow;
  int nrows, roff, part;     // part: -1, or the CTA's partial
};
struct Cut {  // of a CTA: the cut unit that it joins, if its range is the first to start inside one
  int64_t qrow;
  int nrows, cut, first, last;  // pieces: partial `first` of the range before, then partial 0 of the ranges up to `last`
};
struct Misc {
  uint64_t bars[B_COUNT + (B_COUNT & 1)];
  sas::CtaCtl ctl;
  uint32_t tmem;
  int start_b;
  uint32_t sent[2][2];   // loaders of K, of V: tiles whose halves were asked for
  int64_t start_prefix, total;
  int64_t wsum[kThreads / 32];
  uint32_t vmask[3][4];  // rows of tile n that are there, in n % 3
  float red[2][4][MR];   // row maxima of even and odd tiles, by quarter
  Tile ring[kRing];
  uint32_t vis[kRing][kMaxTok][4];  // a published tile's 128 rows: those that each token sees
  Unit units[kUnitSlots];
  Fin fin[2];            // of even and odd units
  uint32_t bits[kMaxTok][kWords];   // coordinator: drafted rows each token of its unit sees
  int16_t parents[kMaxTree];        // coordinator: its request's, -2: not a drafted token's index
  uint4 box[kEpiWarps][128];        // epilogue: 32 rows x 64 bytes per warp
};
constexpr int SMEM_BYTES = OFF_MISC + (int)sizeof(Misc) + 1024;
static_assert(SMEM_BYTES <= 232448, "shared memory over the per-CTA limit");

constexpr size_t kPieceFloats = (size_t)MR * D + 2 * MR;  // O, m (log2 units), l

struct TreeParams {
  const uint8_t* q;
  uint8_t* out;
  float* lse;
  int T, H, G, R, scenario,  // G: head groups of 128, R: pairs of CTAs per group
       K, ratio, win, B, S, layout;
  const int32_t* cu;
  const int32_t* seqused;
  const int32_t* parents;
  const uint8_t* kv[2];  // window pool, compressed pool
  const int32_t* bt[2];
  int bs[2], bt_stride[2];
  int tma[2];            // pages of the pool are copied in boxes of 64 rows
  int64_t nblk[2];
  const int32_t* idx;
  const float* sinks;
  float scale_log2;
  float* part;  // [CTAs][2] pieces
  Cut* cuts;    // [CTAs]
  int32_t* status;
  unsigned long long wait_ns;  // limit of every wait
  CUtensorMap map_kv[2], map_q;
};

// What a request brings: its tokens, and the tiles of each of its units. Units of
// padding alone, after the last token in use, are none of the sequence's (with them
// ranges that hold few used units wait for those that hold many).
struct Req {
  int base, slots, n, used, ctx, thr, lo, units, wtiles, tiles;  // used: tokens up to the last in use, lo: the window tiles' first row
  bool bad;
  __device__ __forceinline__ int64_t all() const { return (int64_t)units * tiles; }
};
__device__ __noinline__ Req request(const TreeParams& p, int b) {
  Req r;
  int n;  // tokens by cu_seqlens_q, from which the append and the decode count the slots, if q has fewer too
  if (p.layout == SAS_LAYOUT_TND) {
    const int c0 = __ldg(p.cu + b), c1 = __ldg(p.cu + b + 1);
    r.base = min(max(c0, 0), p.T);
    r.n = r.slots = max(min(c1, p.T) - r.base, 0);
    n = max(c1 - c0, 0);
  } else {
    r.base = b * p.S;
    r.slots = p.S;
    n = p.cu ? max(__ldg(p.cu + b + 1) - __ldg(p.cu + b), 0) : p.S;
    r.n = min(n, p.S);
  }
  r.ctx = __ldg(p.seqused + b) - n;
  r.bad = r.n > kMaxTree || r.ctx < 0 || r.ctx > kMaxCtx;
  r.thr = p.scenario == 1 || r.bad ? 0 : r.ctx / p.ratio;
  r.used = r.n;
  if (p.layout == SAS_LAYOUT_BSND && !r.bad)  // the last 64 slots are looked through, 8 loads at a time
    for (int k = 0; k < 8 && r.used > 0; ++k) {
      const int from = max(r.used - 8, 0);
      int last = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (from + i < r.used && __ldg(p.parents + r.base + from + i) >= -1) last = from + i + 1;
      r.used = last ? last : from;
      if (last) break;
    }
  const int held = r.bad ? r.slots : r.used;
  r.units = p.scenario == 3 ? held : (int)(((int64_t)held * p.H + UR - 1) / UR);
  r.lo = max(r.ctx - p.win, 0);
  if (p.tma[0]) r.lo &= ~63;
  r.wtiles = r.bad || r.used == 0 ? 1 : (r.ctx - r.lo + r.used + CH - 1) / CH;
  r.tiles = r.wtiles + (r.bad || r.used == 0 ? 0 : p.scenario == 2 ? (r.thr + CH - 1) / CH : p.scenario == 3 && r.thr > 0 ? (p.K + CH - 1) / CH : 0);
  return r;
}
__device__ __forceinline__ int64_t range_start(int64_t total, int R, int r) {
  if (total < (1 << 20)) return (uint32_t)total * (uint32_t)r / (uint32_t)R;  // R <= 2048 here; 64-bit division is slow
  return total * r / R;
}
// CTAs (per head group) that share the sequence; every range has a tile
__device__ __forceinline__ int ranges(int64_t total, int R) { return (int)max((int64_t)1, min((int64_t)R, total)); }

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(sas::smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(sas::smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tma_2d(uint32_t dst, const void* map, uint64_t* bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(sas::smem_u32(bar)), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const void* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(sas::smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// D[tmem of both CTAs] (+)= A B^T over the pair
__device__ __forceinline__ void umma2(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// Arrive on `bar` of both CTAs once every MMA issued before is complete.
__device__ __forceinline__ void commit2(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          sas::smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
// Arrive on `bar` of the pair's first CTA. What it announces is in this CTA's
// shared or tensor memory, written before a proxy or tcgen05 fence of the
// writers, and read there by the pair's MMAs: CTA scope is enough, and a cluster-scope
// release would wait for the warp's global stores too.
__device__ __forceinline__ void arrive_first(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, 0;\n\t"
      "mbarrier.arrive.release.cta.shared::cluster.b64 _, [a];\n\t}" ::"r"(sas::smem_u32(bar))
      : "memory");
}
// Bounded waits, as sas::mbar_wait. Only the first try is inlined: with the
// loops in every place the kernel had 159 KB of code, and its warps, each in
// another part of it, waited for instructions. PAIR: the other CTA's threads
// arrive on the barrier.
template <bool PAIR>
__device__ __forceinline__ bool try_wait(uint64_t* bar, uint32_t parity) {
  if (!PAIR) return sas::mbar_try_wait(bar, parity);
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(sas::smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// A limit that a blocking try could oversleep is met by polls, as there, in a variant
// of the kernel (POLL): a choice at each wait costs 2 to 5% of every call.
__device__ __forceinline__ bool poll_pair(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(sas::smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
template <bool PAIR, bool POLL>
__device__ __noinline__ bool wait_on(uint64_t* bar, uint32_t parity, volatile sas::CtaCtl* ctl, int* status, int where) {
  const uint64_t t0 = sas::globaltimer(), lim = ctl->limit_ns;
  for (uint32_t n = 1;; ++n) {
    if (!POLL ? try_wait<PAIR>(bar, parity) : PAIR ? poll_pair(bar, parity) : sas::mbar_test_wait(bar, parity)) return true;
    if (POLL || (n & 63u) == 0) {
      if (ctl->abort) return false;
      if (sas::globaltimer() - t0 > lim) {
        ctl->abort = 1;
        if (status) atomicCAS(status, 0, SAS_ERR_TIMEOUT_BASE + where);
        return false;
      }
    }
  }
}
template <bool PAIR, bool POLL>
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile sas::CtaCtl* ctl, int* status, int where) {
  return (!POLL && try_wait<PAIR>(bar, parity)) || wait_on<PAIR, POLL>(bar, parity, ctl, status, where);
}
// One lane of the warp. The compiler takes the branch on it as a single
// thread's and keeps MMA operands in uniform registers: 32 products are issued
// in 660 cycles, under `lane == 0` in 1950, which is more than they take to run.
__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
  return e != 0;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void st_shared16(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (DT == SAS_DTYPE_BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return reinterpret_cast<const uint32_t&>(v);
  }
  const __half2 v = __floats2half2_rn(a, b);
  return reinterpret_cast<const uint32_t&>(v);
}
// Two fp32 values in a register pair, and operations on both at once.
__device__ __forceinline__ uint64_t pair(uint32_t a, uint32_t b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(a), "r"(b));
  return v;
}
__device__ __forceinline__ float lo(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t twice(float a) { return pair(__float_as_uint(a), __float_as_uint(a)); }
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ void bad(const TreeParams& p, int code) {
  if (p.status) atomicCAS(p.status, 0, code);
}
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u); }

// The 32 rows from position p0 that a token at position s sees: the cached
// ones of its window, then the drafted ones of its bitmap.
__device__ __noinline__ uint32_t window_bits(int p0, int s, int win, int ctx, const uint32_t* bits) {
  const int c = ctx - p0;  // cached rows before the drafted ones
  uint32_t m = low_bits(c) & ~low_bits(s - win - p0);
  if (c <= 0) {
    const int j = -c, w = j >> 5, o = j & 31;
    if (w < kWords) m = __funnelshift_r(bits[w], w + 1 < kWords ? bits[w + 1] : 0u, o);
  } else if (c < 32) {
    m |= bits[0] << c;
  }
  return m;
}

// Zeroes the half rows [row0, row0 + 32) of a tile's V that hold infinities or NaN.
template <int DT>
__device__ __noinline__ void clear_rows(uint32_t v_base, int row0) {
  constexpr uint32_t ex = DT == SAS_DTYPE_BF16 ? 0x7f80u : 0x7c00u;  // the exponent's bits
#pragma unroll 1
  for (int r = row0; r < row0 + 32; ++r) {
    const uint32_t at = v_base + r * 128;
    uint32_t hot = 0;
#pragma unroll 1
    for (int e = 0; e < 32; ++e) {  // 16-byte pieces
      uint32_t w[4];
      asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at + (e >> 3) * VSLAB + (e & 7) * 16));
#pragma unroll
      for (int x = 0; x < 4; ++x) hot |= ((w[x] & ex) == ex) | (((w[x] >> 16) & ex) == ex);
    }
#pragma unroll 1
    for (int e = 0; hot && e < 32; ++e) st_shared16(at + (e >> 3) * VSLAB + (e & 7) * 16, 0, 0, 0, 0);
  }
}

template <int DT, bool POLL>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) tree_attn_kernel(const __grid_constant__ TreeParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  Misc& ms = *reinterpret_cast<Misc*>(smem + OFF_MISC);
  uint64_t* bars = ms.bars;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int side = blockIdx.x & 1;  // the CTA's place in its pair
  const int g = (blockIdx.x >> 1) % p.G, rank = (blockIdx.x >> 1) / p.G;
  if (tid == 0) {
    auto init = [&](int bar, int n, int count) {
      for (int i = 0; i < n; ++i) sas::mbar_init(&bars[bar + i], count);
    };
    init(B_KFULL, 4, 32 * kLoadWarps);  // and VFULL
    init(B_QFULL, 11, 1);               // QFULL, XK, XV, XQ, KEMPTY, VEMPTY, QEMPTY
    init(B_MASK, 3, kLoadWarps);
    init(B_SFULL, 2, 1);
    init(B_SEMPTY, 3, 2 * kSmWarps);    // and PREADY: softmax warps of both CTAs
    init(B_OFULL, 1, 1);
    init(B_OEMPTY, 3, 2 * kEpiWarps);
    init(B_FIN, 2, kSmWarps);
    init(B_SSYNC, 2, kSmWarps / 2);     // the warps of 32 rows
    init(B_CFULL, kRing, 1);
    init(B_CEMPTY, kRing, 2 * kLoadWarps + 2 + kSmWarps);
    init(B_DRAIN, 2, 1);
    sas::fence_mbar_init();
    ms.ctl.abort = 0;
    ms.ctl.limit_ns = p.wait_ns;
    ms.start_b = p.B;
    ms.start_prefix = 0;
  }
  if (warp == kQkWarp) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sas::smem_u32(&ms.tmem)), "r"(TM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  // every thread takes a run of requests; a block scan of their tiles gives the
  // sequence's length and the request that this CTA's range starts in
  const int per = (p.B + kThreads - 1) / kThreads;
  const int b0 = min(tid * per, p.B), b1 = min(b0 + per, p.B);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) mine += request(p, b).all();
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) ms.wsum[warp] = incl;
  sas::tc_fence_before();
  __syncthreads();
  sas::tc_fence_after();
  int64_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += ms.wsum[w];
    total += ms.wsum[w];
  }
  const int R = ranges(total, p.R);
  const int64_t t0 = rank < R ? range_start(total, R, rank) : total;
  const int64_t t1 = rank < R ? range_start(total, R, rank + 1) : total;
  {
    int64_t at = before + incl - mine;
    for (int b = b0; b < b1; ++b) {
      const int64_t a = per == 1 ? mine : request(p, b).all();
      if (t0 >= at && t0 < at + a) ms.start_b = b, ms.start_prefix = at;
      at += a;
    }
  }
  sas::pdl_launch_dependents();
  sas::tc_fence_before();
  __syncthreads();
  cluster_sync();  // the other CTA's barriers and tensor memory are there
  sas::tc_fence_after();
  const uint32_t tmem = ms.tmem;
  volatile sas::CtaCtl* ctl = &ms.ctl;
  const uint32_t q_base = sas::smem_u32(smem + OFF_Q), k_base = sas::smem_u32(smem + OFF_K),
                 v_base = sas::smem_u32(smem + OFF_V), p_base = sas::smem_u32(smem + OFF_P);
#define WAIT(bar, par, id) wait<false, POLL>(&bars[bar], (par)&1, ctl, p.status, id)
#define WAIT_PAIR(bar, par, id) wait<true, POLL>(&bars[bar], (par)&1, ctl, p.status, id)

  if (warp == kCoordWarp) {
    // ================================================= coordinator
    int b = ms.start_b, cached = -1;
    Req r = request(p, min(b, p.B - 1));
    int64_t prefix = ms.start_prefix, t = t0;
    uint32_t c = 0, uc = 0;
    bool ok = true, lead_cut = false;
    auto publish = [&](int flags, int row0, int nrows, int us) -> bool {
      const int slot = c % kRing;
      if (!__all_sync(0xffffffffu, WAIT(B_CEMPTY + slot, (c / kRing) ^ 1u, W_PUBLISH))) return false;
      if (!(flags & (TF_END | TF_ZERO))) {  // lane: token, 32 rows
        const Unit& un = ms.units[us];
        const int tok = lane >> 2, pos = un.pos[tok];
        uint32_t m = 0;
        if (pos >= 0) m = flags & TF_CMP ? 0xffffffffu : window_bits(row0 + 32 * (lane & 3), pos, p.win, un.ctx, ms.bits[tok]);
        ms.vis[slot][tok][lane & 3] = m;
        __syncwarp();
      }
      if (lane == 0) {
        ms.ring[slot] = Tile{flags, row0, nrows, us};
        sas::mbar_arrive(&bars[B_CFULL + slot]);
      }
      ++c;
      return true;
    };
    while (ok && t < t1 && b < p.B) {
      if (t >= prefix + r.all()) {
        prefix += r.all();
        if (++b < p.B) r = request(p, b);
        continue;
      }
      const int64_t in = t - prefix;
      const int u = in < (1ll << 31) ? (int)((uint32_t)in / (uint32_t)r.tiles) : (int)(in / r.tiles);
      const int64_t ustart = prefix + (int64_t)u * r.tiles, uend = ustart + r.tiles;
      const int k0 = (int)(t - ustart), k1 = (int)min((int64_t)r.tiles, t1 - ustart);
      if (b != cached) {
        __syncwarp();
        if (!r.bad)
          for (int i = lane; i < r.n; i += 32) {
            const int q = __ldg(p.parents + r.base + i);
            ms.parents[i] = (int16_t)(q < -1 ? -2 : min(q, kMaxTree));
          }
        else if (lane == 0 && u == 0 && k0 == 0)
          bad(p, SAS_ERR_BAD_TREE);
        cached = b;
        __syncwarp();
      }
      const int us = uc % kUnitSlots;
      Unit& un = ms.units[us];
      // the unit's rows among the request's, and this CTA's half of them
      const uint32_t H = p.H, first = p.scenario == 3 ? u * H + g * UR : (uint32_t)u * UR;  // T * H < 2^31
      const uint32_t end = p.scenario == 3 ? min(first + UR, (u + 1) * H) : min(first + UR, (uint32_t)r.slots * H);
      const uint32_t row_in = first + side * MR;
      const int nrows = end > row_in ? (int)min((uint32_t)MR, end - row_in) : 0;
      const int i0 = (int)(first / H), i1 = (int)((end - 1) / H);
      const int mine = nrows ? (int)(row_in / H) - i0 : 0;  // this CTA's first token among the unit's
      // the slot's last readers are done: see kUnitSlots; the ring wait below
      // orders this warp's writes after their reads
      if (!__all_sync(0xffffffffu, WAIT(B_CEMPTY + c % kRing, (c / kRing) ^ 1u, W_UNIT_SLOT))) break;
      int pos = -1;
      if (lane < kMaxUnitTok) {
        const int slot = lane - mine;
        uint32_t* bits = slot >= 0 && slot < kMaxTok ? ms.bits[slot] : nullptr;
        const int words = max((min(r.n, kMaxTree) + 31) / 32, 1);
        // window_bits reads up to five words past the last one with a bit
        if (bits)
          for (int w = 0; w < min(words + 5, kWords); ++w) bits[w] = 0;
        const int i = i0 + lane;
        if (i <= i1 && i < r.n && !r.bad && ms.parents[i] >= -1) {
          int j = i, d = 0;
          bool good = true;
          while (true) {
            if (bits && d <= p.win) bits[j >> 5] |= 1u << (j & 31);
            const int q = ms.parents[j];
            if (q == -1) break;
            if (q < -1 || q >= j) {  // after an unused slot, or not before its child
              good = false;
              break;
            }
            j = q;
            ++d;
          }
          if (good) pos = r.ctx + d;
          else bad(p, SAS_ERR_BAD_TREE);
        }
        if (bits) un.pos[slot] = pos;
      }
      if (lane == 0) {
        un.b = b;
        un.tok = r.base + i0;
        un.ctx = r.ctx;
        un.thr = r.thr;
        un.qrow = (int64_t)r.base * p.H + row_in;
        un.nrows = nrows;
        un.roff = (int)(row_in % H);
      }
      __syncwarp();
      const bool any = __any_sync(0xffffffffu, pos >= 0);
      const bool whole = k0 == 0 && k1 == r.tiles;
      if (k0 > 0 && any) {
        lead_cut = true;
        const int64_t before = range_start(total, R, rank - 1);
        int last = rank;  // the range that holds the unit's last tile
        while (last + 1 < R && range_start(total, R, last + 1) < uend) ++last;
        // the first piece is partial 0 of its CTA if the unit starts with that range
        if (lane == 0)
          p.cuts[blockIdx.x] = Cut{(int64_t)r.base * p.H + row_in, nrows, before <= ustart, before == ustart ? 0 : 1, last};
      }
      if (!any) {
        if (k0 == 0) {
          ok = publish(TF_ZERO, 0, 0, us);
          ++uc;
        }
      } else {
        ++uc;
        const int part = whole ? 0 : (t == t0 ? TF_PART0 : TF_PART1);
        const int wrows = r.ctx - r.lo + min(i1, r.used - 1) + 1;  // up to the unit's last drafted token
        for (int k = k0; k < k1 && ok; ++k) {
          int fl = part | (k == k0 ? TF_FIRST : 0) | (k == k1 - 1 ? TF_LAST : 0), row0, n;
          if (k < r.wtiles) {
            row0 = r.lo + k * CH;
            n = min(CH, wrows - k * CH);
          } else {
            row0 = (k - r.wtiles) * CH;
            n = min(CH, (p.scenario == 3 ? p.K : r.thr) - row0);
            fl |= TF_CMP | (p.scenario == 3 ? TF_TOPK : 0);
          }
          ok = publish(fl, row0, max(n, 0), us);
        }
      }
      t = ustart + k1;
    }
    if (lane == 0 && !lead_cut) p.cuts[blockIdx.x].cut = 0;
    if (ok) publish(TF_END, 0, 0, 0);
  } else if (warp >= kKWarp0) {
    // ================================================= loaders
    // By cp.async, warps of K: 16 of this CTA's 64 K rows of a tile each; warps of
    // V: 32 of the tile's 128 rows each, this CTA's 256 columns. By TMA, lane 0 of
    // the first warp does it all. The warps of K also tell which rows are there.
    const bool is_v = warp >= kVWarp0;
    const int lw = (warp - kKWarp0) & 3;
    // K: lanes 0-15 have the warp's K rows, 16-31 the same of the other CTA's half (for the mask)
    const int my_row = is_v ? lw * 32 + lane : (lane < 16 ? side : side ^ 1) * 64 + lw * 16 + (lane & 15);
    const int full = is_v ? B_VFULL : B_KFULL, empty = is_v ? B_VEMPTY : B_KEMPTY;
    uint32_t c = 0, n = 0, q = 0, n0 = 0;  // n, n0: tiles whose second, first half this warp has arrived for
    // pool row of position pos of a request's table, -1: none
    auto lookup = [&](int f, int b, int pos) -> int {
      const int col = pos / p.bs[f];
      const int blk = col < p.bt_stride[f] ? __ldg(p.bt[f] + (int64_t)b * p.bt_stride[f] + col) : 0x7fffffff;
      if (blk >= p.nblk[f]) bad(p, SAS_ERR_BAD_BLOCK_ENTRY);
      return blk < 0 || blk >= p.nblk[f] ? -1 : blk * p.bs[f] + (pos - col * p.bs[f]);
    };
    while (true) {
      if (!__all_sync(0xffffffffu, WAIT(B_CFULL + c % kRing, c / kRing, W_LOAD_TILE))) break;
      const Tile t = ms.ring[c % kRing];
      if (t.flags & TF_END) break;
      if (!(t.flags & TF_ZERO)) {
        const Unit& u = ms.units[t.uslot];
        const int f = (t.flags & TF_CMP) ? 1 : 0;
        const bool tma = p.tma[f] && !(t.flags & TF_TOPK);
        int row = -1;  // pool row of tile row my_row, -1: none (TMA: of the first of lane's 64 rows)
        if (tma) {
          if (lane < 2 && 64 * lane < t.nrows) row = lookup(f, u.b, t.row0 + 64 * lane);
        } else if (my_row < t.nrows) {
          int pos = t.row0 + my_row;
          if (t.flags & TF_TOPK) pos = __ldg(p.idx + (int64_t)u.tok * p.K + pos);
          if (!(t.flags & TF_TOPK) || (pos >= 0 && pos < u.thr)) row = lookup(f, u.b, pos);
        }
        if (!is_v && lw == 0 && (t.flags & TF_FIRST)) {
          if (!__all_sync(0xffffffffu, WAIT(B_QEMPTY, q ^ 1u, W_Q_FREE))) break;
          const int q0 = (int)u.qrow;
          if (elect_one()) {  // rows past the unit's are other rows, or zero past the last: nobody reads their results
            sas::mbar_arrive_expect_tx(&bars[B_QFULL], 8 * QSLAB);
#pragma unroll
            for (int i = 0; i < 8; ++i) tma_2d(q_base + i * QSLAB, &p.map_q, &bars[B_QFULL], i * 64, q0);
          }
          __syncwarp();
          ++q;
        }
        const uint32_t there = __ballot_sync(0xffffffffu, row >= 0);
        // TMA: page and row of the two halves; one without a page is read past the
        // last block, where TMA gives zeros
        const int pg = row < 0 ? (int)p.nblk[f] : row / p.bs[f], at = row < 0 ? 0 : row - pg * p.bs[f];
        const int b0 = __shfl_sync(0xffffffffu, pg, 0), b1 = __shfl_sync(0xffffffffu, pg, 1);
        const int a0 = __shfl_sync(0xffffffffu, at, 0), a1 = __shfl_sync(0xffffffffu, at, 1);
        const CUtensorMap* map = &p.map_kv[f];
        const uint8_t* src = p.kv[f] + lane * 16 + (is_v ? side * 512 : 0);
        // V rows that the product's K steps take; the others stay as they are
        const int cnt = is_v ? min(32, max(16, (t.nrows + 15) & ~15) - lw * 32) : 16;
        bool ok = true;
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          ok = __all_sync(0xffffffffu, WAIT(empty + h, n ^ 1u, is_v ? W_V_FREE : W_K_FREE));
          if (!ok) break;
          if (tma) {
            if (lw == 0 && elect_one()) {
              expect_tx(&bars[full + h], 4 * KSLAB);
              if (is_v) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  const uint32_t dst = v_base + (2 * h + i) * VSLAB;
                  tma_3d(dst, map, &bars[B_VFULL + h], side * 256 + (2 * h + i) * 64, a0, b0);
                  tma_3d(dst + 8192, map, &bars[B_VFULL + h], side * 256 + (2 * h + i) * 64, a1, b1);
                }
              } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  tma_3d(k_base + (4 * h + i) * KSLAB, map, &bars[B_KFULL + h], (4 * h + i) * 64, side ? a1 : a0, side ? b1 : b0);
              }
            }
            __syncwarp();
            sas::mbar_arrive(&bars[full + h]);
          } else if (is_v) {  // 256 bytes of two rows at a time
            const uint32_t dst = v_base + (2 * h + ((lane >> 3) & 1)) * VSLAB + lw * 32 * 128;
#pragma unroll 8  // 2 or 16: 6% slower
            for (int i = 0; i < cnt; i += 2) {
              const int ii = i + (lane >> 4), ri = __shfl_sync(0xffffffffu, row, ii);
              cp16(dst + ii * 128 + (((lane & 7) ^ (ii & 7)) << 4), src + (int64_t)max(ri, 0) * (D * 2) + h * 256 - (lane >> 4) * 256, ri >= 0 ? 16u : 0u);
            }
            cp_arrive(&bars[full + h]);
          } else {
            const uint32_t dst = k_base + (4 * h + (lane >> 3)) * KSLAB + lw * 16 * 128;
#pragma unroll 8
            for (int i = 0; i < 16; ++i) {  // all of them: absent rows are zero, so that their scores are finite
              const int ri = __shfl_sync(0xffffffffu, row, i);
              cp16(dst + i * 128 + (((lane & 7) ^ (i & 7)) << 4), src + (int64_t)max(ri, 0) * (D * 2) + h * 512, ri >= 0 ? 16u : 0u);
            }
            cp_arrive(&bars[full + h]);
          }
          if (h == 0) ++n0;
          if (!is_v && h == 0 && lane == 0) {
            // Tile n - 3's mask was here. It is done with: K came free after the
            // scores of n - 1, for which those of n - 3 had been read, after it.
            if (tma) {
              ms.vmask[n % 3][lw] = (there >> (lw >> 1)) & 1u ? low_bits(t.nrows - 32 * lw) : 0u;
            } else {
              uint16_t* part = reinterpret_cast<uint16_t*>(ms.vmask[n % 3]);
              part[side * 4 + lw] = (uint16_t)there;
              part[(side ^ 1) * 4 + lw] = (uint16_t)(there >> 16);
            }
            sas::mbar_arrive(&bars[B_MASK + n % 3]);
          }
        }
        if (!ok) break;
        ++n;
      }
      __syncwarp();
      if (lane == 0) sas::mbar_arrive(&bars[B_CEMPTY + c % kRing]);
      ++c;
    }
    // No copy may still be landing when the CTA leaves. After a wait that gave up, the
    // warp that issues the boxes may have asked for a half (the first one alone, too) for
    // which another warp has not arrived: each half's last phase then lacks that arrival
    // and never ends. It is one phase at most, as the phase before it had to be complete.
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (lw == 0 && lane == 0) ms.sent[is_v][0] = n0, ms.sent[is_v][1] = n;
    sas::named_bar_sync(1 + is_v, 32 * kLoadWarps);
    for (int h = 0; h < 2; ++h) {
      const uint32_t sent = ms.sent[is_v][h];
      if ((h ? n : n0) < sent) sas::mbar_arrive(&bars[full + h]);
      if (lw == 0 && sent > 0) sas::mbar_wait_drain(&bars[full + h], (sent - 1) & 1, SAS_WAIT_LIMIT_NS);
    }
    if (lw == 0 && !is_v && q > 0) sas::mbar_wait_drain(&bars[B_QFULL], (q - 1) & 1, SAS_WAIT_LIMIT_NS);
  } else if (warp == kQkWarp || warp == kPvWarp) {
    // ================================================= MMA issuers
    if (elect_one()) {
      constexpr int fmt = DT == SAS_DTYPE_BF16 ? 1 : 0;
      const bool pv = warp == kPvWarp;
      auto pass_on = [&](int bar, int to, uint32_t par, int id) -> bool {
        if (!WAIT(bar, par, id)) return false;
        sas::fence_proxy_async_smem();  // cp.async writes -> tensor core reads
        arrive_first(&bars[to]);
        return true;
      };
      uint32_t c = 0, n = 0, u = 0;
      while (true) {
        if (!WAIT(B_CFULL + c % kRing, c / kRing, W_MMA_TILE)) break;
        const Tile t = ms.ring[c % kRing];
        if (t.flags & TF_END) break;
        if (!(t.flags & TF_ZERO)) {
          if (side) {
            if (pv) {
              if (!pass_on(B_VFULL, B_XV, n, W_PASS_V) || !pass_on(B_VFULL + 1, B_XV + 1, n, W_PASS_V)) break;
            } else {
              if ((t.flags & TF_FIRST) && !pass_on(B_QFULL, B_XQ, u++, W_PASS_Q)) break;
              if (!pass_on(B_KFULL, B_XK, n, W_PASS_K) || !pass_on(B_KFULL + 1, B_XK + 1, n, W_PASS_K)) break;
            }
          } else if (pv) {  // O += P V
            constexpr uint32_t id_o = sas::umma_idesc_f16(fmt, UR, 256, 0, 1);
            const uint64_t p_desc = sas::umma_desc_sw128(p_base, 16, 1024), v_desc = sas::umma_desc_sw128(v_base, VSLAB, 1024);
            if (!WAIT_PAIR(B_PREADY, n, W_PV_P)) break;
            const int steps = max(1, (t.nrows + 15) / 16);
            bool ok = true;
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
              const uint32_t oh = 2 * u + h, place = oh % 3;
              ok = (!(t.flags & TF_FIRST) || WAIT_PAIR(B_OEMPTY + place, (oh / 3) ^ 1u, W_PV_O)) && WAIT(B_VFULL + h, n, W_PV_V) &&
                   WAIT_PAIR(B_XV + h, n, W_PV_XV);
              if (!ok) break;
              sas::fence_proxy_async_smem();
              sas::tc_fence_after();
#pragma unroll 1
              for (int ks = 0; ks < steps; ++ks)
                umma2(tmem + TM_O + 128 * place, p_desc + (((ks >> 2) * QSLAB + (ks & 3) * 32) >> 4),
                      v_desc + ((2 * h * VSLAB + ks * 2048) >> 4), id_o, !((t.flags & TF_FIRST) && ks == 0));
              commit2(&bars[B_VEMPTY + h]);
            }
            if (!ok) break;
            if (t.flags & TF_LAST) {
              commit2(&bars[B_OFULL]);
              ++u;
            }
          } else {  // S = Q K^T
            constexpr uint32_t id_s = sas::umma_idesc_f16(fmt, UR, CH, 0, 0);
            const uint64_t q_desc = sas::umma_desc_sw128(q_base, 16, 1024), k_desc = sas::umma_desc_sw128(k_base, 16, 1024);
            if (t.flags & TF_FIRST) {
              if (!WAIT(B_QFULL, u, W_QK_Q) || !WAIT_PAIR(B_XQ, u, W_QK_XQ)) break;
              ++u;
            }
            if (!WAIT_PAIR(B_SEMPTY + (n & 1), (n >> 1) ^ 1u, W_QK_S)) break;
            bool ok = true;
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
              ok = WAIT(B_KFULL + h, n, W_QK_K) && WAIT_PAIR(B_XK + h, n, W_QK_XK);
              if (!ok) break;
              sas::fence_proxy_async_smem();
              sas::tc_fence_after();
#pragma unroll 1
              for (int s = 4 * h; s < 4 * h + 4; ++s)
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                  umma2(tmem + TM_S + 64 * (n & 1), q_desc + ((s * QSLAB + kk * 32) >> 4), k_desc + ((s * KSLAB + kk * 32) >> 4), id_s,
                        (s | kk) != 0);
              commit2(&bars[B_KEMPTY + h]);
            }
            if (!ok) break;
            commit2(&bars[B_SFULL + (n & 1)]);
            if (t.flags & TF_LAST) commit2(&bars[B_QEMPTY]);
          }
          ++n;
        }
        sas::mbar_arrive(&bars[B_CEMPTY + c % kRing]);
        ++c;
      }
      // nothing may still run on TMEM or shared memory when the pair leaves, nor a commit
      // still be on its way to the second CTA's barriers, which so waits for the last one
      if (!side) commit2(&bars[B_DRAIN + pv]);
      sas::mbar_wait_drain(&bars[B_DRAIN + pv], 0, SAS_WAIT_LIMIT_NS);
    }
    __syncwarp();
  } else if (warp >= kEpiWarp0 && warp < kEpiWarp0 + kEpiWarps) {
    // ================================================= epilogue
    // Warp w has TMEM lanes [32 w, + 32): 32 rows, 256 of their columns.
    const int ew = warp - kEpiWarp0, row = (ew & 1) * 32 + lane, ch = ew >> 1;
    const uint32_t tl = tmem + ((uint32_t)ew << 21), box = sas::smem_u32(ms.box[ew]);
    if (p.layout == SAS_LAYOUT_TND) {  // rows that no request holds are zero
      const int et = tid - 32 * kEpiWarp0;
      const int64_t lo = (int64_t)min(max(__ldg(p.cu), 0), p.T) * p.H, hi = (int64_t)min(max(__ldg(p.cu + p.B), 0), p.T) * p.H;
      const int64_t all = (int64_t)p.T * p.H;
      for (int64_t r = blockIdx.x; r < all; r += gridDim.x) {
        if (r >= lo && r < hi) {  // jump over the held rows, staying on this CTA's share
          if (hi == all) break;
          r += (hi - r + gridDim.x - 1) / gridDim.x * gridDim.x - gridDim.x;
          continue;
        }
        if (et < 64) reinterpret_cast<uint4*>(p.out + r * D * 2)[et] = make_uint4(0, 0, 0, 0);
        if (et == 64 && p.lse) p.lse[r] = 0.f;
      }
    }
    if (p.layout == SAS_LAYOUT_BSND)  // and rows of padding alone
      for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
        const Req r = request(p, b);
        const int64_t lo = (int64_t)r.base * p.H + min((int64_t)r.units * (p.scenario == 3 ? p.H : UR), (int64_t)r.slots * p.H);
        const int et = tid - 32 * kEpiWarp0, n = (int)((int64_t)(r.base + r.slots) * p.H - lo);
        for (int64_t i = et; i < (int64_t)n * (D / 8); i += 32 * kEpiWarps) reinterpret_cast<uint4*>(p.out + lo * (D * 2))[i] = make_uint4(0, 0, 0, 0);
        for (int i = et; p.lse && i < n; i += 32 * kEpiWarps) p.lse[lo + i] = 0.f;
      }
    for (uint32_t u = 0;; ++u) {
      if (!__all_sync(0xffffffffu, WAIT(B_FIN + (u & 1), u >> 1, W_EPI_UNIT))) break;
      const Fin& fin = ms.fin[u & 1];
      const int nrows = fin.nrows, part = fin.part;
      if (nrows < 0) break;  // the range is done
      const int64_t qrow = fin.qrow;
      const float m = fin.m[row], l0 = fin.l[0][row];
      const float l = (l0 + fin.l[1][row]) + (fin.l[2][row] + fin.l[3][row]);
      const bool used = !(l0 < 0.f);
      float* const o = p.part + ((size_t)blockIdx.x * 2 + max(part, 0)) * kPieceFloats;
      float k = 0.f;
      if (part >= 0) {
        if (ch == 0) {
          o[MR * D + row] = m;
          o[MR * D + MR + row] = used ? l : -1.f;  // -1: the token is not in use
        }
      } else {
        const float sink = __ldg(p.sinks + (fin.roff + row) % p.H) * kLog2e;
        const float top = fmaxf(m, sink);
        const float a = m == -INFINITY ? 0.f : exp2f(m - top);
        const float den = l * a + (sink == -INFINITY ? 0.f : exp2f(sink - top));
        k = !used || (m == -INFINITY && l == 0.f) ? 0.f : a / den;
        if (row < nrows && ch == 0 && p.lse) p.lse[qrow + row] = used ? (top + log2f(den)) * kLn2 : 0.f;
      }
      if (!__all_sync(0xffffffffu, WAIT(B_OFULL, u, W_EPI_O))) break;
      sas::tc_fence_after();
      const int nr = min(32, nrows - (ew & 1) * 32);
      uint8_t* out = p.out + (qrow + (ew & 1) * 32) * (D * 2) + ch * 512 + (lane & 3) * 16;
      const uint64_t k2 = twice(k);
#pragma unroll 1
      for (int x = 0; x < 8; ++x) {
        uint32_t r[32];
        __syncwarp();
        const uint32_t oh = 2 * u + (x >> 2), place = oh % 3;
        sas::tmem_ld32(tl + TM_O + 128 * place + 32 * (x & 3), r);
        sas::tmem_wait_ld();
        if ((x & 3) == 3) {  // this half of O is read
          sas::tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_first(&bars[B_OEMPTY + place]);
        }
        if (part >= 0) {  // [D / 4][64 rows] of float4: a warp's stores are contiguous
          uint4* d4 = reinterpret_cast<uint4*>(o) + (size_t)(ch * 64 + x * 8) * MR + row;
#pragma unroll
          for (int i = 0; i < 8; ++i) d4[i * MR] = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
        } else {
          // through shared memory, so that a store writes whole sectors of 8 rows
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint64_t y = mul2(pair(r[8 * i + 2 * e], r[8 * i + 2 * e + 1]), k2);
              v[e] = k == 0.f ? 0u : pack2<DT>(lo(y), hi(y));
            }
            st_shared16(box + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4), v[0], v[1], v[2], v[3]);
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int rr = 8 * i + (lane >> 2);
            uint4 q4;
            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(q4.x), "=r"(q4.y), "=r"(q4.z), "=r"(q4.w)
                         : "r"(box + rr * 64 + (((lane & 3) ^ ((rr >> 1) & 3)) << 4)));
            if (rr < nr) *reinterpret_cast<uint4*>(out + (int64_t)rr * (D * 2) + x * 64) = q4;
          }
        }
      }
    }
  } else if (warp < kSmWarps) {
    // ================================================= softmax
    // Warps w and w + 4 share TMEM lanes: thread = row, columns [32 part, + 32)
    // of a tile's 128.
    const int row = (warp & 1) * 32 + lane, ch = (warp >> 1) & 1, gr = warp >> 2, part = 2 * ch + gr;
    const uint32_t tl = tmem + ((uint32_t)(warp & 3) << 21);
    const bool flip = p.scale_log2 < 0.f;
    const float scale = flip ? -p.scale_log2 : p.scale_log2;
    uint32_t c = 0, n = 0, u = 0;
    float m = -INFINITY, l = 0.f;
    int tok = 0;
    bool used = false, ok = true;
    while (ok) {
      if (!__all_sync(0xffffffffu, WAIT(B_CFULL + c % kRing, c / kRing, W_SM_TILE))) break;
      const Tile t = ms.ring[c % kRing];
      if (t.flags & TF_END) {
        // the epilogue ends too; its place is free as below
        if (n > 0 && !__all_sync(0xffffffffu, WAIT(B_VEMPTY + 1, n ^ 1u, W_SM_END))) break;
        ms.fin[u & 1].nrows = -1;
        __syncwarp();
        if (lane == 0) sas::mbar_arrive(&bars[B_FIN + (u & 1)]);
        break;
      }
      const Unit& un = ms.units[t.uslot];
      if (t.flags & TF_ZERO) {
        uint4* o = reinterpret_cast<uint4*>(p.out + un.qrow * (D * 2));
        for (int i = tid; i < un.nrows * (D / 8); i += 32 * kSmWarps) o[i] = make_uint4(0, 0, 0, 0);
        if (p.lse && tid < un.nrows) p.lse[un.qrow + tid] = 0.f;
      } else {
        if (t.flags & TF_FIRST) {
          m = -INFINITY;
          l = 0.f;
          tok = p.scenario == 3 ? 0 : min((un.roff + row) / p.H, kMaxTok - 1);
          used = row < un.nrows && un.pos[tok] >= 0;
        }
        uint32_t see = used ? ms.vis[c % kRing][tok][part] : 0u;
        // rows of the tile that are there, and those that this row's token sees
        ok = __all_sync(0xffffffffu, WAIT(B_MASK + n % 3, n / 3, W_SM_MASK));
        if (!ok) break;
        // rows of the buffers that hold values that some row does not see: stale ones
        // too, past the last of a page's
        const bool check = !(t.flags & TF_CMP) || t.nrows < CH;
        const uint32_t there32 = ms.vmask[n % 3][part];
        see &= there32;
        ok = __all_sync(0xffffffffu, WAIT(B_SFULL + (n & 1), n >> 1, W_SM_S));
        if (!ok) break;
        sas::tc_fence_after();
        uint64_t s[16];
        {
          uint32_t r[32];
          sas::tmem_ld32(tl + TM_S + 64 * (n & 1) + 32 * gr, r);
          sas::tmem_wait_ld();
          sas::tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_first(&bars[B_SEMPTY + (n & 1)]);
          if (flip)
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] ^= 0x80000000u;
          if (check || !__all_sync(0xffffffffu, see == 0xffffffffu)) {
            if (check) {
              // A row may be seen by some tokens only, or by none, and one with
              // infinities or NaN would reach the others' sums as 0 * NaN. All
              // rows' scores with it are not finite, in both CTAs, which their
              // sum shows; each CTA then clears what it holds of such a row's V.
              // A token that sees it has a NaN in l, so its result is NaN.
              uint64_t z[2] = {0, 0};
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                z[0] = add2(z[0], pair(r[i], r[i + 1]));
                z[1] = add2(z[1], pair(r[i + 2], r[i + 3]));
              }
              const float zs = (lo(z[0]) + hi(z[0])) + (lo(z[1]) + hi(z[1]));
              // The tile's V has to be there, after the one before it was done
              // with (its copy alone could be two phases back). A wait that fails
              // shows at the next one.
              if (!(fabsf(zs) < INFINITY) && WAIT(B_VEMPTY + 1, n ^ 1u, W_SM_V_FREE) &&
                  WAIT(B_VFULL, n, W_SM_V) && WAIT(B_VFULL + 1, n, W_SM_V)) {
                clear_rows<DT>(v_base, 32 * part);
                // a score of -inf weighs nothing, but its row is not finite
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (((see >> i) & 1u) && __uint_as_float(r[i]) == -INFINITY) l = NAN;
              }
            }
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!((see >> i) & 1u)) r[i] = 0xff800000u;  // -inf
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = pair(r[2 * i], r[2 * i + 1]);
        }
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = max3(mx, lo(s[i]), hi(s[i]));
        float(*const red)[MR] = ms.red[n & 1];
        red[part][row] = mx;
        __syncwarp();
        if (lane == 0) sas::mbar_arrive(&bars[B_SSYNC + (warp & 1)]);
        ok = __all_sync(0xffffffffu, WAIT(B_SSYNC + (warp & 1), n, W_SM_MAX));
        if (!ok) break;
        mx = fmaxf(fmaxf(red[0][row], red[1][row]), fmaxf(red[2][row], red[3][row])) * scale;
        float fac = 1.f;
        if (mx > m + kMove || (m == -INFINITY && mx > m)) {
          fac = sas::ex2(m - mx);
          m = mx;
          l *= fac;
        }
        const uint64_t sc2 = twice(scale), rf2 = twice(m == -INFINITY ? 0.f : -m);
        uint32_t w[16];
        {
          uint64_t la[2] = {0, 0};
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint64_t x = fma2(s[i], sc2, rf2);
            const float a = sas::ex2(lo(x)), b = sas::ex2(hi(x));
            la[i & 1] = add2(la[i & 1], pair(__float_as_uint(a), __float_as_uint(b)));
            w[i] = pack2<DT>(a, b);
          }
          la[0] = add2(la[0], la[1]);
          l += lo(la[0]) + hi(la[0]);
        }
        // the product before this tile's is complete, and P may be written
        ok = __all_sync(0xffffffffu, WAIT(B_VEMPTY + 1, n ^ 1u, W_SM_P));
        if (!ok) break;
        sas::tc_fence_after();
        if (!(t.flags & TF_FIRST) && __any_sync(0xffffffffu, fac != 1.f)) {
#pragma unroll 1
          for (int x = 0; x < 128; x += 32) {
            const uint32_t at = tl + TM_O + 128 * ((2 * u + gr) % 3) + x;
            uint32_t r[32];
            sas::tmem_ld32(at, r);
            sas::tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * fac);
            sas::tmem_st32(at, r);
          }
          sas::tmem_wait_st();
        }
        const uint32_t pd = p_base + ch * QSLAB + row * 128;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          st_shared16(pd + (((4 * gr + e) ^ (row & 7)) << 4), w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
        sas::fence_proxy_async_smem();
        sas::tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_first(&bars[B_PREADY]);
        ++n;
        if (t.flags & TF_LAST) {
          // The place was unit u - 2's: the first half of its O was read, after
          // these, before the second half of unit u - 1's first product, and that
          // is complete.
          Fin& fin = ms.fin[u & 1];
          fin.l[part][row] = used ? l : -1.f;
          if (part == 0) fin.m[row] = m;
          if (tid == 0) {
            fin.qrow = un.qrow, fin.nrows = un.nrows, fin.roff = un.roff;
            fin.part = t.flags & TF_PART1 ? 1 : t.flags & TF_PART0 ? 0 : -1;
          }
          __syncwarp();
          if (lane == 0) sas::mbar_arrive(&bars[B_FIN + (u & 1)]);
          ++u;
        }
      }
      __syncwarp();
      if (lane == 0) sas::mbar_arrive(&bars[B_CEMPTY + c % kRing]);
      ++c;
    }
  }
  sas::tc_fence_before();
  __syncthreads();
  cluster_sync();  // the other CTA no longer reads this one's shared memory or arrives on it
  if (warp == kQkWarp) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TM_COLS) : "memory");
#undef WAIT
#undef WAIT_PAIR
}

// Joins the pieces of a cut unit, in order: the block of CTA c does so when c's
// range is the first to start inside the unit; blockIdx.y takes 64 columns. A
// thread has 16 columns of a row. All it needs of the two pieces that there are at
// least is asked for at once. For one tile a pair it is a chain of latencies, 3.5 us
// (5 with loads as their values were needed); 38 MB of pieces take 11 us, with 16 to
// 128 columns a block and 3 to 8 blocks an SM alike.
template <int DT>
__global__ void __launch_bounds__(256, 4) tree_combine_kernel(const __grid_constant__ TreeParams p) {
  sas::pdl_wait();
  const int ctas = 2 * p.G;  // of a range
  const int g = blockIdx.x % ctas, rank = blockIdx.x / ctas;
  const Cut c = p.cuts[blockIdx.x];
  if (!c.cut) return;
  auto piece = [&](int r) { return p.part + ((size_t)(r * ctas + g) * 2 + (r == rank - 1 ? c.first : 0)) * kPieceFloats; };
  __shared__ __align__(16) uint8_t tile[MR * 128];
  const int row = threadIdx.x & 63, c4 = (threadIdx.x >> 6) * 4, d4 = blockIdx.y * 16 + c4;
  if (row < c.nrows) {
    struct Part { float m, l; float4 v[4]; };
    auto load = [&](int r) {
      const float* q = piece(r);
      Part x;
      x.m = q[MR * D + row], x.l = q[MR * D + MR + row];
#pragma unroll
      for (int i = 0; i < 4; ++i) x.v[i] = reinterpret_cast<const float4*>(q)[(size_t)(d4 + i) * MR + row];
      return x;
    };
    const Part a = load(rank - 1), b = load(rank);
    const float sink = __ldg(p.sinks + (c.qrow + row) % p.H) * kLog2e;
    float top = fmaxf(sink, fmaxf(a.m, b.m));
    for (int r = rank + 1; r <= c.last; ++r) top = fmaxf(top, piece(r)[MR * D + row]);
    const float base = top == -INFINITY ? 0.f : top;
    float den = exp2f(sink - base);
    float o[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = 0.f;
    const bool used = !(a.l < 0.f);
    auto add = [&](const Part& x) {
      const float w = exp2f(x.m - base);
      den = fmaf(x.l, w, den);
      if (w != 0.f)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          o[4 * i] = fmaf(x.v[i].x, w, o[4 * i]), o[4 * i + 1] = fmaf(x.v[i].y, w, o[4 * i + 1]);
          o[4 * i + 2] = fmaf(x.v[i].z, w, o[4 * i + 2]), o[4 * i + 3] = fmaf(x.v[i].w, w, o[4 * i + 3]);
        }
    };
    add(a);
    add(b);
    for (int r = rank + 1; r <= c.last; ++r) add(load(r));
    const float k = used && (top != -INFINITY || den != den) ? 1.f / den : 0.f;
    uint32_t v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k != 0.f ? pack2<DT>(o[2 * i] * k, o[2 * i + 1] * k) : 0u;
    uint4* to = reinterpret_cast<uint4*>(tile + row * 128 + c4 * 8);
    to[0] = make_uint4(v[0], v[1], v[2], v[3]);
    to[1] = make_uint4(v[4], v[5], v[6], v[7]);
    if (blockIdx.y == 0 && c4 == 0 && p.lse) p.lse[c.qrow + row] = used ? (top + log2f(den)) * kLn2 : 0.f;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < c.nrows * 8; i += 256)
    *reinterpret_cast<uint4*>(p.out + (c.qrow + (i >> 3)) * (D * 2) + blockIdx.y * 128 + (i & 7) * 16) =
        *reinterpret_cast<const uint4*>(tile + (i >> 3) * 128 + (i & 7) * 16);
}

size_t workspace_bytes(int sms) { return (size_t)sms * (sizeof(Cut) + 2 * kPieceFloats * sizeof(float)); }

template <int DT>
int launch(const TreeParams& p, cudaStream_t st) {
  auto kern = p.wait_ns < sas::kPollLimitNs ? tree_attn_kernel<DT, true> : tree_attn_kernel<DT, false>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess) return SAS_ERR_CUDA;
  kern<<<2 * p.R * p.G, kThreads, SMEM_BYTES, st>>>(p);
  if (cudaGetLastError() != cudaSuccess) return SAS_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * p.R * p.G, D / 64);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, tree_combine_kernel<DT>, p) == cudaSuccess ? SAS_OK : SAS_ERR_CUDA;
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
  static EncodeTiled fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiled>(ptr);
  });
  return fn;
}
// Boxes of 64 rows x 64 columns of rows of 512: [outer, rows, 512], or [rows, 512] with outer 0.
bool make_map(CUtensorMap* m, const void* base, int dtype, int64_t outer, int64_t rows) {
  const EncodeTiled enc = encode_tiled();
  if (!enc) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)rows, (cuuint64_t)outer};
  const cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)rows * D * 2};
  const cuuint32_t box[3] = {64, 64, 1}, step[3] = {1, 1, 1};
  return enc(m, dtype == SAS_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, outer ? 3 : 2,
             const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool aligned16(const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; }

}  // namespace

extern "C" {

size_t sas_tree_attn_workspace_bytes(int32_t num_sms) { return num_sms > 0 ? workspace_bytes(num_sms) : 0; }

int sas_tree_attn_sharedkv(const void* q, int32_t T, int32_t H, int32_t head_dim, int32_t dtype, int32_t layout,
                           int32_t B, int32_t S, const int32_t* cu, const int32_t* seqused, const int32_t* parents,
                           const void* ori_kv, int64_t ori_nblk, int32_t ori_bs, const int32_t* ori_bt,
                           int32_t ori_stride, const void* cmp_kv, int64_t cmp_nblk, int32_t cmp_bs,
                           const int32_t* cmp_bt, int32_t cmp_stride, const int32_t* idx, int32_t K,
                           const float* sinks, float softmax_scale, int32_t ratio, int32_t win, int32_t scenario,
                           void* out, float* lse, int32_t num_sms, int32_t* status, void* workspace,
                           size_t workspace_size, void* stream) {
  if (dtype != SAS_DTYPE_BF16 && dtype != SAS_DTYPE_FP16) return SAS_ERR_UNSUPPORTED;
  if (head_dim != D || H <= 0 || H % 8 || T < 0 || B < 0 || win < 0 || num_sms <= 0) return SAS_ERR_INVALID_ARG;
  if (scenario < 1 || scenario > 3) return SAS_ERR_INVALID_ARG;
  if (layout == SAS_LAYOUT_TND ? (!cu && B > 0) : (layout != SAS_LAYOUT_BSND || S < 0 || (int64_t)B * S != T))
    return SAS_ERR_INVALID_ARG;
  if (T == 0) return SAS_OK;
  if (!q || !out || !sinks || !parents || B <= 0 || !seqused || !ori_kv || !ori_bt || ori_bs <= 0 || ori_stride <= 0 || ori_nblk < 0)
    return SAS_ERR_INVALID_ARG;
  if (scenario >= 2 && (!cmp_kv || !cmp_bt || cmp_bs <= 0 || cmp_stride <= 0 || cmp_nblk < 0 || ratio <= 0))
    return SAS_ERR_INVALID_ARG;
  if (scenario == 3 && (!idx || K <= 0)) return SAS_ERR_INVALID_ARG;
  if (!aligned16(q) || !aligned16(out) || !aligned16(ori_kv) || !aligned16(cmp_kv)) return SAS_ERR_INVALID_ARG;
  if (!workspace || workspace_size < workspace_bytes(num_sms)) return SAS_ERR_WORKSPACE;
  if (!sas::select_device_of(q)) return SAS_ERR_CUDA;
  TreeParams p = {};
  p.q = static_cast<const uint8_t*>(q);
  p.out = static_cast<uint8_t*>(out);
  p.lse = lse;
  p.T = T, p.H = H, p.scenario = scenario, p.K = K, p.ratio = ratio, p.win = win < kMaxCtx ? win : kMaxCtx, p.B = B, p.S = S, p.layout = layout;
  p.G = scenario == 3 ? (H + UR - 1) / UR : 1;
  if (2 * p.G > num_sms) return SAS_ERR_UNSUPPORTED;
  p.R = num_sms / (2 * p.G);
  p.cu = cu, p.seqused = seqused, p.parents = parents;
  p.kv[0] = static_cast<const uint8_t*>(ori_kv), p.kv[1] = static_cast<const uint8_t*>(cmp_kv);
  p.bt[0] = ori_bt, p.bt[1] = cmp_bt;
  p.bs[0] = ori_bs, p.bs[1] = cmp_bs;
  p.bt_stride[0] = ori_stride, p.bt_stride[1] = cmp_stride;
  p.nblk[0] = ori_nblk, p.nblk[1] = cmp_nblk;
  p.idx = idx, p.sinks = sinks, p.scale_log2 = softmax_scale == 0.f ? 1e-30f : softmax_scale * kLog2e;  // 0 * -inf would not mask
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.part = reinterpret_cast<float*>(ws);
  p.cuts = reinterpret_cast<Cut*>(ws + (size_t)num_sms * 2 * kPieceFloats * sizeof(float));
  p.status = status;
  p.wait_ns = sas::wait_limit_ns();
  if ((int64_t)T * H >= (1ll << 31)) return SAS_ERR_UNSUPPORTED;
  if (!make_map(&p.map_q, q, dtype, 0, (int64_t)T * H)) return SAS_ERR_CUDA;
  for (int f = 0; f < (scenario == 2 ? 2 : 1); ++f) {
    p.tma[f] = p.bs[f] % 64 == 0 && p.nblk[f] > 0;
    if (p.tma[f] && !make_map(&p.map_kv[f], p.kv[f], dtype, p.nblk[f], p.bs[f])) return SAS_ERR_CUDA;
  }
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == SAS_DTYPE_BF16 ? launch<SAS_DTYPE_BF16>(p, st) : launch<SAS_DTYPE_FP16>(p, st);
}

}  // extern "C"
