// Gradient of attention with a sliding window and sink tokens (sm_100a,
// tcgen05): dQ, dK, dV from dO, the inputs and the forward's O and
// log-sum-exp L.
//
//   P  = exp(scale Q K^T - L)        delta = sum_d dO * O
//   dV = P^T dO                      dS = P * (dO V^T - delta)
//   dQ = scale dS K                  dK = scale dS^T Q
// with dK and dV summed over the query heads of a kv head.
//
// Three kernels: the rows' statistics (memory bound), one persistent kernel
// that first works through the key tiles (dK, dV) and then through the query
// tiles (dQ), and, where sink keys are seen from behind their window, a small
// one that joins their partial sums (see kv_piece).  The scores are computed
// for the key tiles and again for the query tiles (7 products in place of 5),
// because each sum then has one owner and a fixed order: no atomics on values,
// equal inputs give equal bits, and no fp32 copy of dQ goes through memory.
// P and dS are rounded to the inputs' type as MMA operands; every sum is fp32
// in TMEM.
//
// Roles of the persistent kernel, one CTA per SM:
//   warp 0     TMA of the item's first own tile (K or Q), of ring A (Q or K)
//              and of the row statistics
//   warp 3     TMA of the second own tile (V or dO) and of ring B (dO or V)
//   warp 1     MMA issuer
//   warp 2     TMEM owner; takes work items from a counter and works them out
//   warps 4-11  elementwise: thread = TMEM lane, 64 of a tile's 128 columns
//   warps 12-15 read an item's sums out of TMEM and store them, while the
//               elementwise warps go on with the next item (when they did it
//               themselves, every item began some 4000 cycles later)
// Ring A is three tiles deep and ring B two (with D = 128 that fills shared
// memory): a tile of A is needed by the last product of a step and again
// missing at the first product of the next but one, so with two slots the
// MMA warp waited 2000 cycles per step for it.
#include <algorithm>

#include "attn_ops.cuh"

namespace gpo {

constexpr int kGradA = 3, kGradB = 2;  // ring depths
constexpr int kGradThreads = 512;      // 4 service, 8 elementwise, 4 storing warps
constexpr int kGradEwWarps = 8, kGradOutWarps = 4;
// 512 threads launch at 128 registers; an elementwise thread needs 168.
constexpr int kGradLowRegs = 88, kGradEwRegs = 168, kGradOutRegs = 88;
static_assert(128 * kGradLowRegs + 256 * kGradEwRegs + 128 * kGradOutRegs <= 128 * kGradThreads,
              "register split exceeds the launch's registers");
constexpr int kGradReaders = 3 + kGradEwWarps + kGradOutWarps;  // of an item: all but warp 2

struct GradArgs {
  AttnGeom geom;
  // per packed row: -L in the log2 domain, and -delta; 128 + 128 floats per
  // (batch, kv head, query tile)
  float* stats;
  // sums of dK and dV rows of sink keys that several CTAs share
  float* partial;
  const void *out, *dout;
  const float* lse;
  void *dq, *dk, *dv;
  int64_t o_batch, o_token, o_head, do_batch, do_token, do_head;
  int64_t dq_batch, dq_token, dq_head, dk_batch, dk_token, dk_head, dv_batch, dv_token, dv_head;
  float scale, scale_log2;
  int sink_tiles;  // key tiles with a sink key; 0: nothing to join
  int far_tiles;   // query tiles of a far piece (see kv_piece)
  int far_pieces;  // far pieces of a sink tile
  int blind;               // first tokens, which see no key
  int kv_items, items;     // items [0, kv_items): key tiles, then query tiles
  unsigned int* next;      // counter of items, zeroed by the statistics kernel
  bool wide_dq, wide_dkv;  // rows on 32 bytes
  unsigned int* err;
};

__device__ __forceinline__ float* grad_stats(const GradArgs& a, int b, int h, int tile) {
  return a.stats + ((static_cast<int64_t>(b) * a.geom.heads_kv + h) * a.geom.tiles + tile) * 256;
}

// ---------------------------------------------------------------- row stats
// One block per (query tile, kv head, batch); D / 8 lanes read a row of O
// and dO as 16-byte vectors.  O is the forward's, rounded to the inputs' type:
// its part in delta is off by up to u sum_d |dO| |O|.  Rows of many keys do not
// feel it; where rows see a few, dS is a small difference and dQ, dK are up to
// 2.3 times as far from the exact gradient as their own rounding (bf16 4.2e-3
// against 1.8e-3).  The exact delta is a sum over P and dP, which would take
// two more products (9 in place of 7) before the first dS.
template <typename T, int D>
__global__ void __launch_bounds__(256) attn_grad_stats_kernel(const GradArgs a) {
  const AttnGeom& g = a.geom;
  let_next_start();
  wait_for_previous();
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.next = 0u;
  if (g.tiles == 0) return;
  constexpr int LPR = D / 8, RPW = 32 / LPR;  // lanes per row, rows per warp
  const int tile = blockIdx.x % g.tiles, bh = blockIdx.x / g.tiles;
  const int h = bh % g.heads_kv, b = bh / g.heads_kv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* st = grad_stats(a, b, h, tile);
#pragma unroll 4
  for (int r0 = warp * 16; r0 < warp * 16 + 16; r0 += RPW) {
    const int r = r0 + lane / LPR;
    const int token = tile * g.tpt + r / g.g, head = h * g.g + r % g.g;
    const bool live = r < g.tpt * g.g && token < g.q_len && token >= a.blind;
    float s = 0.f, l = 0.f;
    if (live) {
      if (lane % LPR == 0)
        l = a.lse[(static_cast<int64_t>(b) * g.q_len + token) *
                      (static_cast<int64_t>(g.heads_kv) * g.g) + head];
      const uint4 x = *reinterpret_cast<const uint4*>(
          static_cast<const T*>(a.out) + b * a.o_batch + token * a.o_token + head * a.o_head +
          (lane % LPR) * 8);
      const uint4 y = *reinterpret_cast<const uint4*>(
          static_cast<const T*>(a.dout) + b * a.do_batch + token * a.do_token +
          head * a.do_head + (lane % LPR) * 8);
      const T* xe = reinterpret_cast<const T*>(&x);
      const T* ye = reinterpret_cast<const T*>(&y);
#pragma unroll
      for (int i = 0; i < 8; ++i) s += Elem<T>::to_f(xe[i]) * Elem<T>::to_f(ye[i]);
    }
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane % LPR == 0) {
      float nl = -INFINITY;  // no query in this row: P is 0
      if (live) {
        // a row whose scores were all -inf has P = 0 everywhere, too
        nl = l == -INFINITY ? -INFINITY : -l * 1.4426950408889634f;
      }
      st[r] = nl;
      st[128 + r] = live ? -s : 0.f;
    }
  }
}

// ------------------------------------------------------------- shared parts
struct KvPiece {
  int b, h, kt, piece;  // piece 0: main
  int first, n;         // query tiles
};

struct QItem {
  int b, h, t0, t1, tile;
  AttnSeq seq;
  AttnBlocks blk;
};

// A work item as warp 2 hands it to the other roles.
struct GradWork {
  int kind;  // 0: none left, 1: key tile, 2: query tile
  int n;     // steps
  KvPiece p;
  QItem q;
};

struct GradShared {
  uint64_t own_full[2], own_empty[2];
  uint64_t a_full[kGradA], a_empty[kGradA];
  uint64_t a_raw[kGradA];  // K copied, to be cleared before a_full (grad_clears)
  uint64_t a_cleared;      // the storing warps' parts of it
  uint64_t b_full[kGradB], b_empty[kGradB];
  uint64_t st_full[2], st_empty[2];  // row statistics (key tiles)
  uint64_t s_full, dp_full;          // S of key tiles; dP
  uint64_t q_s_full[2];              // the two S buffers of query tiles
  uint64_t p_ready, ds_ready;
  uint64_t sum_full[2], sum_free[2];  // dV; dK or dQ
  uint64_t item_full[2], item_empty[2];
  uint64_t drain;
  GradWork work[2];
  uint32_t tmem_base;
  int abort;
};

template <int D>
struct GradGeom {
  static constexpr uint32_t TILE = 128u * D * 2;  // bytes of a 128-row tile
  static constexpr uint32_t OWN = 0;
  static constexpr uint32_t RING_A = 2 * TILE;
  static constexpr uint32_t RING_B = RING_A + kGradA * TILE;
  static constexpr uint32_t STATS = RING_B + kGradB * TILE;
  static constexpr uint32_t SHARED = STATS + 2 * 1024u;
  static constexpr uint32_t BYTES = SHARED + sizeof(GradShared);
  static_assert(BYTES <= kMaxSmemPerCta, "shared memory");
};

__device__ __forceinline__ void grad_init(GradShared& sh) {
  auto init = [](uint64_t* b, int n, uint32_t count) {
    for (int i = 0; i < n; ++i) mbar_init(smem_u32(b + i), count);
  };
  init(sh.own_full, 2, 1);
  init(sh.own_empty, 2, 1);
  init(sh.a_full, kGradA, 1);
  init(sh.a_empty, kGradA, 1);
  init(sh.a_raw, kGradA, 1);
  init(&sh.a_cleared, 1, kGradOutWarps);
  init(sh.b_full, kGradB, 1);
  init(sh.b_empty, kGradB, 1);
  init(sh.st_full, 2, 1);
  init(sh.st_empty, 2, kGradEwWarps);
  init(&sh.s_full, 1, 1);
  init(&sh.dp_full, 1, 1);
  init(sh.q_s_full, 2, 1);
  init(&sh.p_ready, 1, kGradEwWarps);
  init(&sh.ds_ready, 1, kGradEwWarps);
  init(sh.sum_full, 2, 1);
  init(sh.sum_free, 2, kGradOutWarps);
  init(sh.item_full, 2, 1);
  init(sh.item_empty, 2, kGradReaders);
  init(&sh.drain, 1, 1);
  sh.abort = 0;
  fence_barrier_init();
}

// Whether rows of a K block of ring A are cleared before the MMAs read it:
// keys that no token sees hold anything, and 0 * NaN is not 0 in dS K.  The copy
// of such a block ends at a_raw; the storing warps clear it and announce
// a_full, so that no other role has a part in it.  UNSEEN instances alone
// (attn_has_unseen).
__device__ __forceinline__ bool grad_clears(const AttnGeom& g, const QItem& q, int key0) {
  return key0 < attn_unseen(g, q.seq) && attn_unseen_rows(g, q.seq, key0).any();
}

template <int N>
struct GradRing {
  int slot = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void step() {
    if (++slot == N) {
      slot = 0;
      parity ^= 1u;
    }
  }
};

// The CTA's it-th item for one role; false when there is none (or the wait
// failed).
template <bool WARP>
__device__ __forceinline__ bool grad_take(GradShared& sh, uint32_t& it, GradWork& w,
                                          unsigned int* err, uint32_t site, bool& ok) {
  const int i = it & 1u;
  ok = mbar_wait(smem_u32(&sh.item_full[i]), (it >> 1) & 1u, &sh.abort, err, site);
  if (WARP) ok = __all_sync(0xffffffffu, ok);
  if (!ok) return false;
  w = sh.work[i];
  if (WARP) __syncwarp();
  if (!WARP || (threadIdx.x & 31) == 0) mbar_arrive(smem_u32(&sh.item_empty[i]));
  ++it;
  return w.kind != 0;
}

// D[tmem, 128 x N] (+)= A B^T over 128-byte-swizzled K-major tiles of 128
// rows and D dims (both operands in shared memory).
template <int D>
__device__ __forceinline__ void mma_rows(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo,
                                         uint32_t idesc) {
  constexpr uint64_t HI = smem_desc_hi(8 * 128, 128);
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    const uint32_t off = ((kk / 4) * 128 * 128 + (kk % 4) * 32) >> 4;
    mma_f16_ss(d_tmem, HI | (a_lo + off), HI | (b_lo + off), idesc, kk > 0 ? 1u : 0u);
  }
}
// D[tmem, 128 x D] += A B with A 128 x 128 in TMEM (16-bit pairs; columns
// 64 .. 127 start at column 64 of the region) and B 128 rows x D dims.
__device__ __forceinline__ void mma_cols(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo,
                                         uint32_t idesc, bool first) {
  constexpr uint64_t HI = smem_desc_hi(8 * 128, 128);
#pragma unroll
  for (int kk = 0; kk < 8; ++kk)
    mma_f16_ts(d_tmem, a_tmem + (kk / 4) * 64 + (kk % 4) * 8,
               HI | (b_lo + ((kk * 16 * 128) >> 4)), idesc, (first && kk == 0) ? 0u : 1u);
}

template <int FMT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return FMT == 1 ? pack_bf16(lo, hi) : pack_f16(lo, hi);
}

// One row of N fp32 TMEM columns, times `f`, to N 16-bit elements at dst.
template <typename T, int FMT, int N>
__device__ __forceinline__ void store_row(uint32_t taddr, T* dst, float f, bool live, bool zero,
                                          bool wide) {
#pragma unroll
  for (int c = 0; c < N / 32; ++c) {
    uint32_t r[32];
    tmem_ld32(taddr + c * 32, r);
    tmem_wait_ld();
    if (!live) continue;
    uint32_t pk[16];
#pragma unroll
    for (int i = 0; i < 16; ++i)
      pk[i] = zero ? 0u : pack2<FMT>(__uint_as_float(r[2 * i]) * f,
                                     __uint_as_float(r[2 * i + 1]) * f);
    store_pairs8(dst + c * 32, pk, wide);
    store_pairs8(dst + c * 32 + 16, pk + 8, wide);
  }
}

// ------------------------------------------------------------------ dK, dV
// Key tile kt is seen by the query tiles [first, last].  For a tile with
// sink keys these are: the tiles of its window (the main piece), and all
// later ones, which see the sink keys alone; those are cut into far pieces
// of far_tiles query tiles, so that no CTA has a longer way than the others.
// The pieces' sums of the sink rows are joined by attn_grad_join_kernel.
__device__ __forceinline__ void kv_tile_range(const GradArgs& a, int kt, int& first, int& last) {
  const AttnGeom& g = a.geom;
  const int off = g.kv_len - g.q_len;
  const int k0 = kt * 128, k1 = min(k0 + 127, g.kv_len - 1);
  const int t_lo = max(0, k0 - off);
  const int t_hi = g.window == kOpsNoWindow ? g.q_len - 1
                                            : min(g.q_len - 1, k1 - off + g.window - 1);
  first = t_lo / g.tpt;
  last = t_hi < t_lo ? first - 1 : t_hi / g.tpt;
}

__device__ __forceinline__ KvPiece kv_piece(const GradArgs& a, int item) {
  const AttnGeom& g = a.geom;
  const int heads = g.heads_kv * g.batch;
  const int r = item / heads, bh = item % heads;
  KvPiece p;
  p.h = bh % g.heads_kv;
  p.b = bh / g.heads_kv;
  const int far = a.sink_tiles * a.far_pieces;
  p.kt = r < far ? r / a.far_pieces : r - far;
  int first, last;
  kv_tile_range(a, p.kt, first, last);
  if (r < far) {
    p.piece = 1 + r % a.far_pieces;
    p.first = max(last + 1, first) + (p.piece - 1) * a.far_tiles;
    p.n = max(0, min(a.far_tiles, g.tiles - p.first));
  } else {
    p.piece = 0;
    p.first = first;
    p.n = max(0, last - first + 1);
  }
  return p;
}

// Row `key` of piece `piece` in the partial sums: dV and then dK, D floats each.
template <int D>
__device__ __forceinline__ float* kv_partial(const GradArgs& a, int b, int h, int key, int piece) {
  const int64_t row = (static_cast<int64_t>(b) * a.geom.heads_kv + h) * a.geom.sinks + key;
  return a.partial + (row * (1 + a.far_pieces) + piece) * (2 * D);
}

// ------------------------------------------------------------ query tiles
__device__ __forceinline__ QItem q_item(const GradArgs& a, int item) {
  const AttnGeom& g = a.geom;
  QItem it;
  const int r = (item - a.kv_items) / g.heads_kv;
  it.h = (item - a.kv_items) % g.heads_kv;
  it.b = r % g.batch;
  it.tile = g.tiles - 1 - r / g.batch;  // the longest rows first
  it.seq = AttnSeq{g.q_len, g.kv_len, 0, g.kv_len - g.q_len};
  it.t0 = it.tile * g.tpt;
  it.t1 = min(it.t0 + g.tpt, g.q_len);
  it.blk = attn_blocks(g, it.seq, it.t0, it.t1);
  return it;
}

// Warp 2: takes an item once every role has begun the one before, and not
// earlier: an item that waits in a busy CTA is one that an idle CTA lacks.
__device__ __forceinline__ void grad_schedule(const GradArgs& args, GradShared& sh) {
  for (int it = 0;; ++it) {
    if (it >= 1 && !mbar_wait(smem_u32(&sh.item_empty[(it - 1) & 1]), ((it - 1) >> 1) & 1u,
                              &sh.abort, args.err, kErrWaitProducer))
      return;
    const unsigned int item = atomicAdd(args.next, 1u);
    GradWork w{};
    if (item < static_cast<unsigned int>(args.items)) {
      if (item < static_cast<unsigned int>(args.kv_items)) {
        w.kind = 1;
        w.p = kv_piece(args, static_cast<int>(item));
        w.n = w.p.n;
      } else {
        w.kind = 2;
        w.q = q_item(args, static_cast<int>(item));
        w.n = w.q.blk.n;
      }
    }
    sh.work[it & 1] = w;
    mbar_arrive(smem_u32(&sh.item_full[it & 1]));
    if (w.kind == 0) return;
  }
}

template <int N>
__device__ __forceinline__ void grad_regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void grad_regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

struct GradMaps {
  const CUtensorMap *q, *dout, *k, *v;
};

// ---------------------------------------------------------------- producers
// Side 0: own tile K (key tiles) or Q, ring A of Q + statistics, or of K.
// Side 1: own tile V or dO, ring B of dO or V.
template <int D, int SIDE, bool UNSEEN>
__device__ __forceinline__ void grad_producer(const GradArgs& args, GradShared& sh,
                                              const GradMaps& maps, uint32_t base) {
  using G = GradGeom<D>;
  constexpr int N = SIDE == 0 ? kGradA : kGradB;
  const AttnGeom& g = args.geom;
  unsigned int* err = args.err;
  volatile int* abort_flag = &sh.abort;
  const uint32_t own_smem = base + G::OWN + SIDE * G::TILE;
  const uint32_t ring = base + (SIDE == 0 ? G::RING_A : G::RING_B);
  uint64_t* full = SIDE == 0 ? sh.a_full : sh.b_full;
  uint64_t* empty = SIDE == 0 ? sh.a_empty : sh.b_empty;
  const uint32_t rows_bytes = static_cast<uint32_t>(g.tpt * g.g) * D * 2;
  auto wait = [&](const uint64_t* bar, uint32_t parity) {
    return mbar_wait(smem_u32(bar), parity, abort_flag, err, kErrWaitProducer);
  };
  // 128 keys from `row`, or the rows of a query tile.  Tokens that see no key
  // may hold anything: the maps of Q and dO begin behind them, and what a copy
  // asks for in front of a map arrives as zeros.
  uint32_t raw = 0, raw_parity = 0;  // bit s: slot s's last copy ends at a_raw; its parity
  auto load_keys = [&](uint32_t dst, const CUtensorMap* m, uint64_t* bar, int h, int row, int b) {
    mbar_arrive_expect_tx(smem_u32(bar), G::TILE);
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
      tma_load_4d(dst + c * 128 * 128, m, smem_u32(bar), c * 64, h, row, b);
  };
  auto load_rows = [&](uint32_t dst, const CUtensorMap* m, uint64_t* bar, int h, int token,
                       int b) {
    mbar_arrive_expect_tx(smem_u32(bar), rows_bytes);
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
      tma_load_5d(dst + c * 128 * 128, m, smem_u32(bar), c * 64, 0, h, token - args.blind, b);
  };
  bool ok = true;
  int own = 0, issued = 0, stats = 0;
  GradRing<N> pos;
  GradRing<2> st;
  uint32_t taken = 0;
  GradWork w;
  while (grad_take<false>(sh, taken, w, err, kErrWaitProducer, ok)) {
    const bool keys = w.kind == 1;
    const KvPiece& p = w.p;
    const QItem& qi = w.q;
    const int n = w.n;
    if (n == 0) continue;
    if (own > 0 && !wait(&sh.own_empty[SIDE], (own - 1) & 1u)) {
      ok = false;
      break;
    }
    if (keys)
      load_keys(own_smem, SIDE == 0 ? maps.k : maps.v, &sh.own_full[SIDE], p.h, p.kt * 128, p.b);
    else
      load_rows(own_smem, SIDE == 0 ? maps.q : maps.dout, &sh.own_full[SIDE], qi.h, qi.t0, qi.b);
    ++own;
    // the row statistics of a query tile, or of every query tile of a key tile
    auto load_stats = [&](int b, int h, int tile) {
      if (!wait(&sh.st_empty[st.slot], st.parity ^ 1u)) return false;
      const uint32_t bar = smem_u32(&sh.st_full[st.slot]);
      mbar_arrive_expect_tx(bar, 1024u);
      bulk_load(base + G::STATS + st.slot * 1024u, grad_stats(args, b, h, tile), 1024u, bar);
      ++stats;
      st.step();
      return true;
    };
    if (SIDE == 0 && !keys && !load_stats(qi.b, qi.h, qi.tile)) {
      ok = false;
      break;
    }
    for (int j = 0; j < n; ++j) {
      if (!wait(&empty[pos.slot], pos.parity ^ 1u)) {
        ok = false;
        break;
      }
      const uint32_t dst = ring + pos.slot * G::TILE, bit = 1u << pos.slot;
      if (UNSEEN) raw &= ~bit;
      if (keys) {
        load_rows(dst, SIDE == 0 ? maps.q : maps.dout, &full[pos.slot], p.h,
                  (p.first + j) * g.tpt, p.b);
      } else {
        const int key0 = qi.blk.at(j) * 128;
        uint64_t* bar = &full[pos.slot];
        if (UNSEEN && SIDE == 0 && grad_clears(g, qi, key0)) {
          bar = &sh.a_raw[pos.slot];
          raw |= bit;
          raw_parity ^= bit;
        }
        load_keys(dst, SIDE == 0 ? maps.k : maps.v, bar, qi.h, key0, qi.b);
      }
      ++issued;
      pos.step();
      if (SIDE == 0 && keys && !load_stats(p.b, p.h, p.first + j)) {
        ok = false;
        break;
      }
    }
    if (!ok) break;
  }
  if (!ok) {
    // let the copies in flight land before the CTA can exit
    if (own > 0) mbar_wait_drain(smem_u32(&sh.own_full[SIDE]), (own - 1) & 1u, err);
    for (int j = max(0, issued - N); j < issued; ++j) {
      const int at = j % N;
      if (UNSEEN && ((raw >> at) & 1u))  // raw_parity has turned once more than the phase it waits for
        mbar_wait_drain(smem_u32(&sh.a_raw[at]), ((raw_parity >> at) & 1u) ^ 1u, err);
      else
        mbar_wait_drain(smem_u32(&full[at]), (j / N) & 1u, err);
    }
    for (int j = max(0, stats - 2); j < stats; ++j)
      mbar_wait_drain(smem_u32(&sh.st_full[j & 1]), (j >> 1) & 1u, err);
  }
}

// -------------------------------------------------------------- MMA issuer
// Key tiles: S(j+1) follows dV(j), which reads P(j) in the same columns, and
// dP(j+1) follows dK(j) in the same way: MMAs run in issue order.
// Query tiles: S(j+1) goes to the other buffer before dS(j) is waited for;
// dP(j+1) then has its columns back and comes before dQ(j), so that the
// elementwise warps wait least.
template <int D>
struct GradTmem {
  // key tiles: S^T and P^T, dP^T and dS^T, dV, dK
  static constexpr uint32_t S = 0, DP = 128, DV = 256, DK = 256 + D;
  // query tiles: two S buffers (dS overlays S), dP, dQ
  static constexpr uint32_t QS = 0, QDP = 256, DQ = 384;
};

template <int FMT, int D>
__device__ __forceinline__ void grad_mma(const GradArgs& args, GradShared& sh, uint32_t base,
                                         uint32_t tmem) {
  using G = GradGeom<D>;
  using C = GradTmem<D>;
  constexpr uint32_t IDESC_S = make_idesc(FMT, 128, 128, false, false);
  constexpr uint32_t IDESC_O = make_idesc(FMT, 128, D, false, true);
  unsigned int* err = args.err;
  volatile int* abort_flag = &sh.abort;
  auto wait = [&](const uint64_t* bar, uint32_t parity) {
    const uint32_t b = smem_u32(bar);
    return mbar_test_wait(b, parity) || mbar_wait(b, parity, abort_flag, err, kErrWaitMma);
  };
  auto commit = [&](const uint64_t* bar) { mma_commit(smem_u32(bar)); };
  const uint32_t own0 = smem_desc_lo(base + G::OWN, 16);
  const uint32_t own1 = smem_desc_lo(base + G::OWN + G::TILE, 16);
  // descriptors of a ring tile as rows (K-major) and as columns (MN-major)
  auto rows_of = [&](uint32_t ring, int slot) {
    return smem_desc_lo(base + ring + slot * G::TILE, 16);
  };
  auto cols_of = [&](uint32_t ring, int slot) {
    return smem_desc_lo(base + ring + slot * G::TILE, 128 * 128);
  };
  bool ok = true, was_keys = true;
  GradRing<kGradA> a;  // next tile of ring A that has not been waited for
  GradRing<kGradB> b;
  uint32_t own = 0, kown = 0, cnt = 0, qcnt = 0;
  uint32_t taken = 0;
  GradWork w;
  while (grad_take<false>(sh, taken, w, err, kErrWaitMma, ok)) {
    const bool keys = w.kind == 1;
    const int n = w.n;
    if (n == 0) continue;
    const uint32_t op = own & 1u;
    if (keys) {
      ok = wait(&sh.own_full[0], op) && wait(&sh.a_full[a.slot], a.parity);
      if (!ok) break;
      mma_rows<D>(tmem + C::S, own0, rows_of(G::RING_A, a.slot), IDESC_S);
      commit(&sh.s_full);
      if (n == 1) commit(&sh.own_empty[0]);
      ok = wait(&sh.own_full[1], op) && wait(&sh.b_full[b.slot], b.parity);
      if (!ok) break;
      mma_rows<D>(tmem + C::DP, own1, rows_of(G::RING_B, b.slot), IDESC_S);
      commit(&sh.dp_full);
      if (n == 1) commit(&sh.own_empty[1]);
      for (int j = 0; j < n && ok; ++j, ++cnt) {
        const int aj = a.slot, bj = b.slot;
        const bool more = j + 1 < n;
        ok = wait(&sh.p_ready, cnt & 1u);
        // the previous item's dV has been read out of TMEM
        if (ok && j == 0 && own > 0) ok = wait(&sh.sum_free[0], (own - 1) & 1u);
        if (!ok) break;
        tc_fence_after();
        mma_cols(tmem + C::DV, tmem + C::S, cols_of(G::RING_B, bj), IDESC_O, j == 0);
        commit(&sh.b_empty[bj]);
        if (!more) commit(&sh.sum_full[0]);
        a.step();
        b.step();
        if (more) {
          ok = wait(&sh.a_full[a.slot], a.parity);
          if (!ok) break;
          mma_rows<D>(tmem + C::S, own0, rows_of(G::RING_A, a.slot), IDESC_S);
          commit(&sh.s_full);
          if (j + 2 == n) commit(&sh.own_empty[0]);
        }
        ok = wait(&sh.ds_ready, cnt & 1u);
        if (ok && j == 0 && own > 0) ok = wait(&sh.sum_free[1], (own - 1) & 1u);
        if (!ok) break;
        tc_fence_after();
        mma_cols(tmem + C::DK, tmem + C::DP, cols_of(G::RING_A, aj), IDESC_O, j == 0);
        commit(&sh.a_empty[aj]);
        if (more) {
          ok = wait(&sh.b_full[b.slot], b.parity);
          if (!ok) break;
          mma_rows<D>(tmem + C::DP, own1, rows_of(G::RING_B, b.slot), IDESC_S);
          commit(&sh.dp_full);
          if (j + 2 == n) commit(&sh.own_empty[1]);
        } else {
          commit(&sh.sum_full[1]);
        }
      }
      if (ok) ++kown;
    } else {
      ok = wait(&sh.own_full[0], op) && wait(&sh.a_full[a.slot], a.parity);
      if (!ok) break;
      mma_rows<D>(tmem + C::QS + (qcnt & 1u) * 128, own0, rows_of(G::RING_A, a.slot), IDESC_S);
      commit(&sh.q_s_full[qcnt & 1u]);
      if (n == 1) commit(&sh.own_empty[0]);
      ok = wait(&sh.own_full[1], op) && wait(&sh.b_full[b.slot], b.parity);
      // dP of query tiles has the columns of dV (and dK) of key tiles
      const bool turn = was_keys && kown > 0;
      if (ok && turn)
        ok = wait(&sh.sum_free[0], (kown - 1) & 1u) && wait(&sh.sum_free[1], (own - 1) & 1u);
      if (!ok) break;
      was_keys = false;
      mma_rows<D>(tmem + C::QDP, own1, rows_of(G::RING_B, b.slot), IDESC_S);
      commit(&sh.dp_full);
      commit(&sh.b_empty[b.slot]);
      b.step();
      if (n == 1) commit(&sh.own_empty[1]);
      for (int j = 0; j < n && ok; ++j, ++cnt, ++qcnt) {
        const int aj = a.slot;
        const bool more = j + 1 < n;
        a.step();
        if (more) {
          ok = wait(&sh.a_full[a.slot], a.parity);
          if (!ok) break;
          mma_rows<D>(tmem + C::QS + ((qcnt + 1) & 1u) * 128, own0, rows_of(G::RING_A, a.slot),
                      IDESC_S);
          commit(&sh.q_s_full[(qcnt + 1) & 1u]);
          if (j + 2 == n) commit(&sh.own_empty[0]);
        }
        ok = wait(&sh.ds_ready, cnt & 1u);
        if (!ok) break;
        tc_fence_after();
        if (more) {
          ok = wait(&sh.b_full[b.slot], b.parity);
          if (!ok) break;
          mma_rows<D>(tmem + C::QDP, own1, rows_of(G::RING_B, b.slot), IDESC_S);
          commit(&sh.dp_full);
          commit(&sh.b_empty[b.slot]);
          b.step();
          if (j + 2 == n) commit(&sh.own_empty[1]);
        }
        // the previous item's dQ has been read out of TMEM
        if (j == 0 && own > 0 && !turn) {
          ok = wait(&sh.sum_free[1], (own - 1) & 1u);
          if (!ok) break;
          tc_fence_after();
        }
        mma_cols(tmem + C::DQ, tmem + C::QS + (qcnt & 1u) * 128, cols_of(G::RING_A, aj), IDESC_O,
                 j == 0);
        commit(&sh.a_empty[aj]);
        if (!more) commit(&sh.sum_full[1]);
      }
    }
    if (!ok) break;
    ++own;
  }
  if (!ok) {
    mma_commit(smem_u32(&sh.drain));
    mbar_wait_drain(smem_u32(&sh.drain), 0, err);
  }
}

// ------------------------------------------------------------- elementwise
template <typename T, int FMT, int D>
struct GradEw {
  const GradArgs& args;
  GradShared& sh;
  uint32_t base, tmem;
  int wg, row, lane;
  uint32_t lane_addr;
  bool ok = true;
  GradRing<2> st;
  uint32_t cnt = 0, qcnt = 0;  // steps, steps of query tiles

  __device__ __forceinline__ bool wait(const uint64_t* bar, uint32_t parity) {
    return ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, &sh.abort, args.err,
                                                  kErrWaitSoftmax));
  }
  // after TMEM stores that a later MMA reads
  __device__ __forceinline__ void release(uint64_t* bar) {
    tmem_wait_st();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(bar));
  }
  __device__ __forceinline__ void load64(uint32_t taddr, float (&x)[64]) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
      tmem_ld32(taddr + c * 32, *reinterpret_cast<uint32_t(*)[32]>(
                                    reinterpret_cast<uint32_t*>(x) + c * 32));
    tmem_wait_ld();
  }
  // P of a pair.  The exponentials keep the special function unit busy for
  // 1024 cycles per step (16 a cycle).  With D = 64 that is what a step waits
  // for, and every other pair of two runs on the FMA pipe (backward of 8192
  // tokens, W 1024: 454 -> 402 us); with D = 128 a step waits for its MMAs,
  // and the same exchange gained nothing (476 -> 473 us).
  static constexpr int kFma = D == 64 ? 2 : 0;  // of 4 pairs
  static __device__ __forceinline__ void exp2_to(float (&pr)[64], int i, float2 x) {
    float2 y;
    if ((i / 2) % 4 < kFma)
      y = exp2_fma<FMT == 1 ? 3 : 4>(x);
    else
      y = make_float2(ex2_approx(x.x), ex2_approx(x.y));
    pr[i] = y.x;
    pr[i + 1] = y.y;
  }
  // dS = P * (dP - delta) of a pair
  static __device__ __forceinline__ uint32_t ds_pair(const float (&pr)[64], int i,
                                                     const uint32_t (&dp)[32], int k, float2 nd) {
    const float2 d = __fadd2_rn(make_float2(__uint_as_float(dp[k]), __uint_as_float(dp[k + 1])), nd);
    const float2 s = __fmul2_rn(make_float2(pr[i], pr[i + 1]), d);
    return pack2<FMT>(s.x, s.y);
  }
  static __device__ __forceinline__ void mask_pairs(uint32_t (&pk)[32], const uint32_t (&see)[2]) {
#pragma unroll
    for (int i = 0; i < 32; ++i) pk[i] &= pair_mask(see[i / 16], i % 16);
  }

  // thread = key; 64 packed query rows of the tile
  __device__ __forceinline__ void keys(const KvPiece& p) {
    using G = GradGeom<D>;
    using C = GradTmem<D>;
    const AttnGeom& g = args.geom;
    const uint32_t s_t = tmem + lane_addr + C::S + wg * 64;
    const uint32_t dp_t = tmem + lane_addr + C::DP + wg * 64;
    const float2 scale2 = make_float2(args.scale_log2, args.scale_log2);
    const int off = g.kv_len - g.q_len;
    const int k0 = p.kt * 128, key = k0 + row;
    // tokens that see this key: [key - off, key - off + window), or all
    // later ones for a sink key
    const int tok_lo = key - off;
    const int tok_hi = (g.window == kOpsNoWindow || key < g.sinks) ? kOpsMaxLen
                                                                    : tok_lo + g.window - 1;
    for (int j = 0; j < p.n; ++j, ++cnt) {
      const int ta = (p.first + j) * g.tpt, tb = ta + g.tpt - 1;
      // some key of the tile misses some token of the query tile
      const bool masked = k0 + 127 - off > ta ||
                          (g.window != kOpsNoWindow && k0 - off + g.window - 1 < tb);
      // packed rows of this thread's half that see the key: [c_lo, c_hi)
      const int c_lo = (max(tok_lo, ta) - ta) * g.g - wg * 64;
      const int c_hi = (min(tok_hi, tb) - ta + 1) * g.g - wg * 64;
      const uint32_t see[2] = {bits_below(c_hi, 0) & ~bits_below(c_lo, 0),
                               bits_below(c_hi, 1) & ~bits_below(c_lo, 1)};
      if (!wait(&sh.st_full[st.slot], st.parity) || !wait(&sh.s_full, cnt & 1u)) return;
      if (masked && __all_sync(0xffffffffu, (see[0] | see[1]) == 0u)) {
        // no key of this warp is seen by its rows (behind the window of a
        // tile whose sinks are): P and dS are 0
        uint32_t zero[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) zero[i] = 0u;
        tc_fence_after();
        tmem_st32(s_t, zero);
        release(&sh.p_ready);
        if (!wait(&sh.dp_full, cnt & 1u)) return;
        tc_fence_after();
        tmem_st32(dp_t, zero);
        release(&sh.ds_ready);
        if (lane == 0) mbar_arrive(smem_u32(&sh.st_empty[st.slot]));
        st.step();
        continue;
      }
      tc_fence_after();
      const uint32_t stat = base + G::STATS + st.slot * 1024u + wg * 256;
      float pr[64];
      load64(s_t, pr);
#pragma unroll
      for (int i = 0; i < 64; i += 4) {
        float4 nl;
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(nl.x), "=f"(nl.y), "=f"(nl.z), "=f"(nl.w)
                     : "r"(stat + i * 4));
        exp2_to(pr, i, __ffma2_rn(make_float2(pr[i], pr[i + 1]), scale2,
                                  make_float2(nl.x, nl.y)));
        exp2_to(pr, i + 2, __ffma2_rn(make_float2(pr[i + 2], pr[i + 3]), scale2,
                                      make_float2(nl.z, nl.w)));
      }
      {
        uint32_t pk[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) pk[i] = pack2<FMT>(pr[2 * i], pr[2 * i + 1]);
        // masked after packing (two values per operation, whatever they are)
        if (masked) mask_pairs(pk, see);
        tmem_st32(s_t, pk);
      }
      release(&sh.p_ready);
      if (!wait(&sh.dp_full, cnt & 1u)) return;
      tc_fence_after();
      uint32_t pk[32];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t dp[32];
        tmem_ld32(dp_t + c * 32, dp);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          float4 dl;
          asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(dl.x), "=f"(dl.y), "=f"(dl.z), "=f"(dl.w)
                       : "r"(stat + 512 + (c * 32 + i) * 4));
          pk[c * 16 + i / 2] = ds_pair(pr, c * 32 + i, dp, i, make_float2(dl.x, dl.y));
          pk[c * 16 + i / 2 + 1] = ds_pair(pr, c * 32 + i + 2, dp, i + 2, make_float2(dl.z, dl.w));
        }
      }
      if (masked) mask_pairs(pk, see);
      tmem_st32(dp_t, pk);
      release(&sh.ds_ready);
      if (lane == 0) mbar_arrive(smem_u32(&sh.st_empty[st.slot]));
      st.step();
    }
  }

  // thread = packed query row; 64 keys of the block
  __device__ __forceinline__ void rows(const QItem& it) {
    using C = GradTmem<D>;
    const AttnGeom& g = args.geom;
    const uint32_t dp_t = tmem + lane_addr + C::QDP + wg * 64;
    const float2 scale2 = make_float2(args.scale_log2, args.scale_log2);
    const int token = it.t0 + row / g.g;
    if (it.blk.n == 0) return;
    if (!wait(&sh.st_full[st.slot], st.parity)) return;
    float nl, nd;
    {
      const uint32_t stat = base + GradGeom<D>::STATS + st.slot * 1024u + row * 4;
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(nl) : "r"(stat));
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(nd) : "r"(stat + 512));
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&sh.st_empty[st.slot]));
    st.step();
    const float2 shift2 = make_float2(nl, nl), delta2 = make_float2(nd, nd);
    for (int j = 0; j < it.blk.n; ++j, ++cnt, ++qcnt) {
      const int key0 = it.blk.at(j) * 128;
      const bool masked = block_is_masked(g, it.seq, it.t0, it.t1, key0);
      const RowMask rm = row_mask(g, token + it.seq.off, key0 + wg * 64);
      const uint32_t s_t = tmem + lane_addr + C::QS + (qcnt & 1u) * 128 + wg * 64;
      if (!wait(&sh.q_s_full[qcnt & 1u], (qcnt >> 1) & 1u)) return;
      tc_fence_after();
      float pr[64];
      load64(s_t, pr);
#pragma unroll
      for (int i = 0; i < 64; i += 2) {
        exp2_to(pr, i, __ffma2_rn(make_float2(pr[i], pr[i + 1]), scale2, shift2));
      }
      if (!wait(&sh.dp_full, cnt & 1u)) return;
      tc_fence_after();
      uint32_t pk[32];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t dp[32];
        tmem_ld32(dp_t + c * 32, dp);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; i += 2)
          pk[c * 16 + i / 2] = ds_pair(pr, c * 32 + i, dp, i, delta2);
      }
      if (masked) {
        const uint32_t see[2] = {rm.word(0), rm.word(1)};
        mask_pairs(pk, see);
      }
      tmem_st32(s_t, pk);
      release(&sh.ds_ready);
    }
  }
};

// ---------------------------------------------------------- sums to memory
// Thread = TMEM lane: a key's dV and dK, or a query row's dQ.  Before, K blocks
// of a query tile are cleared where no token sees their keys (grad_clears).
template <typename T, int FMT, int D, bool UNSEEN>
__device__ __forceinline__ void grad_out(const GradArgs& args, GradShared& sh, uint32_t base,
                                         uint32_t tmem, int quarter, int lane) {
  using C = GradTmem<D>;
  const AttnGeom& g = args.geom;
  const int row = quarter * 32 + lane;
  const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
  const int row_token = row / g.g, row_head = row % g.g;
  bool ok = true;
  uint32_t taken = 0, own = 0, kown = 0;
  auto wait = [&](const uint64_t* bar, uint32_t parity) {
    ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, &sh.abort, args.err,
                                           kErrWaitEpilogue));
    if (ok) tc_fence_after();
    return ok;
  };
  auto release = [&](uint64_t* bar) {
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(bar));
  };
  // tiles of ring A so far; bit s: parity of slot s's a_raw; blocks cleared
  uint32_t steps = 0, raw_parity = 0, cleared = 0;
  auto clear = [&](const QItem& it, int j) {
    const int key0 = it.blk.at(j) * 128, slot = (steps + j) % kGradA;
    if (!grad_clears(g, it, key0)) return true;
    if (!wait(&sh.a_raw[slot], (raw_parity >> slot) & 1u)) return false;
    raw_parity ^= 1u << slot;
    const AttnUnseenRows u = attn_unseen_rows(g, it.seq, key0);
    const uint32_t tile = base + GradGeom<D>::RING_A + slot * GradGeom<D>::TILE;
    auto rows = [&](int r0, int r1) {
      for (int i = row; i < (r1 - r0) * (D / 8); i += kGradOutWarps * 32) {
        const int r = r0 + i / (D / 8), x = i % (D / 8);
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                         tile + x / 8 * 128 * 128 + r * 128 + x % 8 * 16),
                     "r"(0)
                     : "memory");
      }
    };
    rows(u.a0, u.a1);
    rows(u.b0, u.b1);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&sh.a_cleared));
    if (quarter == 0) {
      if (!wait(&sh.a_cleared, cleared & 1u)) return false;
      if (lane == 0) mbar_arrive(smem_u32(&sh.a_full[slot]));
    }
    ++cleared;
    return true;
  };
  GradWork w;
  while (grad_take<true>(sh, taken, w, args.err, kErrWaitEpilogue, ok)) {
    if (UNSEEN && w.kind == 2)
      for (int j = 0; j < w.n; ++j)
        if (!clear(w.q, j)) return;
    if (UNSEEN) steps += w.n;
    if (w.kind == 1) {
      const KvPiece& p = w.p;
      const int key = p.kt * 128 + row;
      const bool there = key < g.kv_len, sink = args.sink_tiles > 0 && key < g.sinks;
#pragma unroll 1
      for (int m = 0; m < 2; ++m) {
        if (w.n > 0 && !wait(&sh.sum_full[m], (m == 0 ? kown : own) & 1u)) return;
        const uint32_t acc = tmem + lane_addr + (m == 0 ? C::DV : C::DK);
        const float f = m == 0 ? 1.f : args.scale;
        if (p.kt < args.sink_tiles) {
          float* part = sink ? kv_partial<D>(args, p.b, p.h, key, p.piece) + m * D : nullptr;
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t r[32];
            tmem_ld32(acc + c * 32, r);
            tmem_wait_ld();
            if (sink && there) {
#pragma unroll
              for (int i = 0; i < 32; i += 4)
                *reinterpret_cast<float4*>(part + c * 32 + i) =
                    w.n == 0 ? make_float4(0.f, 0.f, 0.f, 0.f)
                             : make_float4(__uint_as_float(r[i]) * f,
                                           __uint_as_float(r[i + 1]) * f,
                                           __uint_as_float(r[i + 2]) * f,
                                           __uint_as_float(r[i + 3]) * f);
            }
          }
        }
        T* dst = m == 0 ? static_cast<T*>(args.dv) + p.b * args.dv_batch + key * args.dv_token +
                              p.h * args.dv_head
                        : static_cast<T*>(args.dk) + p.b * args.dk_batch + key * args.dk_token +
                              p.h * args.dk_head;
        if (p.piece == 0)
          store_row<T, FMT, D>(acc, dst, f, there && !sink, w.n == 0, args.wide_dkv);
        if (w.n > 0) release(&sh.sum_free[m]);
      }
      if (w.n > 0) ++kown;
    } else {
      const QItem& it = w.q;
      const int token = it.t0 + row_token;
      if (w.n > 0 && !wait(&sh.sum_full[1], own & 1u)) return;
      T* dst = static_cast<T*>(args.dq) + it.b * args.dq_batch + token * args.dq_token +
               (it.h * g.g + row_head) * args.dq_head;
      store_row<T, FMT, D>(tmem + lane_addr + C::DQ, dst, args.scale,
                           row_token < g.tpt && token < it.t1, w.n == 0, args.wide_dq);
      if (w.n > 0) release(&sh.sum_free[1]);
    }
    if (w.n > 0) ++own;
  }
}

template <typename T, int FMT, int D, bool UNSEEN>
__global__ void __launch_bounds__(kGradThreads, 1)
    attn_grad_kernel(const __grid_constant__ CUtensorMap tma_q,
                     const __grid_constant__ CUtensorMap tma_do,
                     const __grid_constant__ CUtensorMap tma_k,
                     const __grid_constant__ CUtensorMap tma_v,
                     const __grid_constant__ GradArgs args) {
  using G = GradGeom<D>;
  extern __shared__ __align__(1024) uint8_t dyn_smem[];
  const uint32_t base = smem_u32(dyn_smem);
  GradShared& sh = *reinterpret_cast<GradShared*>(dyn_smem + G::SHARED);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const AttnGeom& g = args.geom;
  if (base & 1023u) {  // the swizzled tiles need the alignment asked for above
    if (threadIdx.x == 0) atomicOr(args.err, kErrBadLaunch);
    return;
  }
  const GradMaps maps{&tma_q, &tma_do, &tma_k, &tma_v};
  if (threadIdx.x == 0) {
    grad_init(sh);
    tma_prefetch_desc(&tma_q);
    tma_prefetch_desc(&tma_do);
    tma_prefetch_desc(&tma_k);
    tma_prefetch_desc(&tma_v);
  }
  // Rows of a query tile that hold no query (128 is not a multiple of g): no
  // copy writes them, and 0 * (what was there) need not be 0.  Cleared in
  // the slots that hold query tiles as dK's and dV's operands (key tiles;
  // query tiles come later and have their rows as the M dimension).
  {
    const int unused = 128 - g.tpt * g.g;
    const int vecs = unused * 8 * (D / 64);
    for (int i = threadIdx.x; i < (kGradA + kGradB) * vecs; i += kGradThreads) {
      const int e = i % vecs, atom = e / (unused * 8), x = e % (unused * 8);
      asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                       base + G::RING_A + (i / vecs) * G::TILE + atom * 128 * 128 +
                       (128 - unused) * 128 + x * 16),
                   "r"(0)
                   : "memory");
    }
    fence_proxy_async_smem();
  }
  if (warp == 2) {
    tmem_alloc(smem_u32(&sh.tmem_base), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem_base;
  let_next_start();
  wait_for_previous();
  if (warp < 4) {
    grad_regs_dec<kGradLowRegs>();
    if (warp == 0) {
      if (elect_one()) grad_producer<D, 0, UNSEEN>(args, sh, maps, base);
    } else if (warp == 1) {
      if (elect_one()) grad_mma<FMT, D>(args, sh, base, tmem);
    } else if (warp == 2) {
      if (elect_one()) grad_schedule(args, sh);
    } else {
      if (elect_one()) grad_producer<D, 1, UNSEEN>(args, sh, maps, base);
    }
  } else if (warp < 12) {
    grad_regs_inc<kGradEwRegs>();
    const int q = warp & 3;
    GradEw<T, FMT, D> ew{args, sh, base, tmem, (warp - 4) >> 2, q * 32 + lane, lane,
                         static_cast<uint32_t>(q * 32) << 16};
    uint32_t taken = 0;
    GradWork w;
    while (grad_take<true>(sh, taken, w, args.err, kErrWaitSoftmax, ew.ok)) {
      if (w.kind == 1)
        ew.keys(w.p);
      else
        ew.rows(w.q);
      if (!ew.ok) break;
    }
  } else {
    grad_regs_dec<kGradOutRegs>();
    grad_out<T, FMT, D, UNSEEN>(args, sh, base, tmem, warp & 3, lane);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2) tmem_dealloc(tmem, 512);
}

// Sum of a sink key's pieces, in their order.
template <typename T, int D>
__global__ void __launch_bounds__(2 * D) attn_grad_join_kernel(const GradArgs a) {
  const AttnGeom& g = a.geom;
  let_next_start();
  wait_for_previous();
  const int key = blockIdx.x % g.sinks, bh = blockIdx.x / g.sinks;
  const int h = bh % g.heads_kv, b = bh / g.heads_kv;
  const int x = threadIdx.x;
  float s = 0.f;
  for (int p = 0; p <= a.far_pieces; ++p) s += kv_partial<D>(a, b, h, key, p)[x];
  T* dst = x < D ? static_cast<T*>(a.dv) + b * a.dv_batch + key * a.dv_token + h * a.dv_head + x
                 : static_cast<T*>(a.dk) + b * a.dk_batch + key * a.dk_token + h * a.dk_head +
                       (x - D);
  *dst = Elem<T>::from_f(s);
}

// ------------------------------------------------------------------- host
namespace {

struct GradPlan {
  int kv_tiles, sink_tiles, far_tiles, far_pieces;
  uint64_t stats_bytes, partial_bytes;  // behind 256 bytes for the item counter
};

GradPlan grad_plan(const AttnGeom& g, int dim) {
  GradPlan p{};
  p.kv_tiles = static_cast<int>(cdiv(g.kv_len, 128));
  if (g.window != kOpsNoWindow && g.sinks > 0) {
    p.sink_tiles = static_cast<int>(cdiv(std::min(g.sinks, g.kv_len), 128));
    // query tiles behind the window of key tile 0, in pieces as long as a
    // key tile's window is
    const int64_t off = g.kv_len - g.q_len;
    const int64_t t_hi = std::min<int64_t>(
        g.q_len - 1, std::min<int64_t>(127, g.kv_len - 1) - off + g.window - 1);
    const int64_t t_lo = std::max<int64_t>(0, -off);
    const int64_t next = std::max<int64_t>(t_hi < t_lo ? t_lo / g.tpt : t_hi / g.tpt + 1, 0);
    p.far_tiles = static_cast<int>((static_cast<int64_t>(g.window) + 128) / g.tpt + 1);
    // Without a later tile there is nothing to join (3 x 250 tokens, W 100:
    // 18.0 -> 16.3 us).  One or two later tiles are far pieces all the same: in
    // the main piece they took longer than the join (3 x 333: 18.7 / 19.5).
    if (next >= g.tiles)
      p.sink_tiles = 0;
    else
      p.far_pieces = static_cast<int>(cdiv(g.tiles - next, p.far_tiles));
  }
  const uint64_t heads = static_cast<uint64_t>(g.batch) * g.heads_kv;
  p.stats_bytes = heads * g.tiles * 1024u;
  p.partial_bytes = p.sink_tiles ? heads * g.sinks * (1u + p.far_pieces) * 2u * dim * 4u : 0u;
  return p;
}

template <typename T, int FMT, int D>
gpo_status run_grad(const AttnProblem& p, const AttnGradProblem& gp, const LaunchCtx& c) {
  const AttnGeom& g = p.geom;
  CUtensorMap mq, mdo, mk, mv;
  // (kv_len = 0: nothing is loaded, and the maps stay whole)
  const int blind = g.kv_len > 0 ? std::max(0, g.q_len - g.kv_len) : 0;
  auto seeing = [&](HeadsView t) {
    t.ptr = static_cast<const char*>(t.ptr) + blind * t.s_token * 2;
    t.tokens -= blind;
    return t;
  };
  if (!encode_rows_map(&mq, p.dtype, seeing(p.q), D, g.g, g.tpt) ||
      !encode_rows_map(&mdo, p.dtype, seeing(gp.dout), D, g.g, g.tpt) ||
      !encode_keys_map(&mk, p.dtype, p.k, D, 128) || !encode_keys_map(&mv, p.dtype, p.v, D, 128))
    return GPO_BAD_ARGS;
  const GradPlan pl = grad_plan(g, D);
  GradArgs a{};
  a.geom = g;
  char* work = static_cast<char*>(gp.workspace);
  a.next = reinterpret_cast<unsigned int*>(work);
  a.stats = reinterpret_cast<float*>(work + 256);
  a.partial = reinterpret_cast<float*>(work + 256 + pl.stats_bytes);
  a.out = gp.out.ptr;
  a.dout = gp.dout.ptr;
  a.lse = gp.lse;
  a.dq = const_cast<void*>(gp.dq.ptr);
  a.dk = const_cast<void*>(gp.dk.ptr);
  a.dv = const_cast<void*>(gp.dv.ptr);
  auto strides = [](const HeadsView& v, int64_t& sb, int64_t& st, int64_t& sh) {
    sb = v.s_batch;
    st = v.s_token;
    sh = v.s_head;
  };
  strides(gp.out, a.o_batch, a.o_token, a.o_head);
  strides(gp.dout, a.do_batch, a.do_token, a.do_head);
  strides(gp.dq, a.dq_batch, a.dq_token, a.dq_head);
  strides(gp.dk, a.dk_batch, a.dk_token, a.dk_head);
  strides(gp.dv, a.dv_batch, a.dv_token, a.dv_head);
  a.wide_dq = rows_on_32(gp.dq);
  a.wide_dkv = rows_on_32(gp.dk) && rows_on_32(gp.dv);
  a.scale = p.scale;
  a.scale_log2 = p.scale * 1.4426950408889634f;
  a.sink_tiles = pl.sink_tiles;
  a.far_tiles = pl.far_tiles;
  a.far_pieces = pl.far_pieces;
  a.blind = blind;
  a.err = c.err;
  const int64_t heads = static_cast<int64_t>(g.batch) * g.heads_kv;
  const int64_t q_items = heads * g.tiles;
  const int64_t kv_items = heads * (pl.kv_tiles + static_cast<int64_t>(pl.sink_tiles) * pl.far_pieces);
  const int64_t most = (1ll << 31) - 1024;
  if (q_items + kv_items > most || heads * g.sinks > most) return GPO_BAD_ARGS;
  a.kv_items = static_cast<int>(kv_items);
  a.items = static_cast<int>(q_items + kv_items);
  if (a.items == 0) return GPO_OK;
  const int sms = c.sm_count > 0 ? c.sm_count : 148;
  gpo_status s = launch_in_order(attn_grad_stats_kernel<T, D>,
                                 static_cast<unsigned>(std::max<int64_t>(1, q_items)), 256, 0,
                                 c.stream, a);
  if (s != GPO_OK) return s;
  auto kern = attn_has_unseen(g) ? attn_grad_kernel<T, FMT, D, true>
                                 : attn_grad_kernel<T, FMT, D, false>;
  constexpr uint32_t dyn = GradGeom<D>::BYTES;
  static_assert(dyn > kOpsAloneBytes, "two CTAs fit an SM");
  s = ensure_smem_attr(reinterpret_cast<const void*>(kern), dyn);
  if (s != GPO_OK) return s;
  s = launch_in_order(kern, static_cast<unsigned>(std::min(a.items, sms)), kGradThreads, dyn,
                      c.stream, mq, mdo, mk, mv, a);
  if (s != GPO_OK || pl.sink_tiles == 0) return s;
  return launch_in_order(attn_grad_join_kernel<T, D>, static_cast<unsigned>(heads * g.sinks), 2 * D,
                         0, c.stream, a);
}

}  // namespace

uint64_t attn_grad_workspace(const AttnProblem& p) {
  const GradPlan pl = grad_plan(p.geom, p.dim);
  return 256u + pl.stats_bytes + pl.partial_bytes;
}

gpo_status launch_attn_grad(const AttnProblem& p, const AttnGradProblem& gp, const LaunchCtx& c) {
  if (p.dtype == GPO_BFLOAT16)
    return p.dim == 128 ? run_grad<__nv_bfloat16, 1, 128>(p, gp, c)
                        : run_grad<__nv_bfloat16, 1, 64>(p, gp, c);
  return p.dim == 128 ? run_grad<__half, 0, 128>(p, gp, c) : run_grad<__half, 0, 64>(p, gp, c);
}

}  // namespace gpo
