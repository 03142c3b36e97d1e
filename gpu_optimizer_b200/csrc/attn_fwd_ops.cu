// Attention with a sliding window and sink tokens over grouped heads, from
// strided dense K/V or from a paged cache (sm_100a, tcgen05).
//
// O = softmax(scale * Q K^T over the visible keys) V and, per row, the
// log-sum-exp of its scaled scores.  One pass over the visible K/V blocks
// with the running maximum and sum of each row in registers.
//
// A unit of work is a span of TILES tiles of 128 query rows of one sequence
// and kv head (attn_ops.cuh: a tile packs all query heads of the kv head,
// so K/V is read once for all of them).  One persistent CTA per SM:
//   warp 0     TMA of Q and of the K ring
//   warp 3     TMA of the V ring; clears V rows of keys that no row may weigh
//   warp 1     MMA issuer; P overlays S in TMEM as 16-bit pairs
//   warp 2     TMEM owner; walks the CTA's stretches and hands them out; sends
//              staged tiles of O to memory
//   warps 4-7  softmax and epilogue of tile 0, thread = query row = TMEM
//   warps 8-11 lane; of tile 1
// TILES = 2 (more than 128 rows per sequence and kv head, more than two tiles
// per SM): both tiles share every K/V block; the issuer alternates them, so
// that one tile's softmax hides behind the other's MMAs.  TILES = 1 (single
// tokens, short chunks): bound by the K/V bytes; three S buffers let S run two
// blocks ahead of PV.
//
// With TILES = 2 a whole tile of O leaves through a staging tile in shared
// memory and TMA.  (Stores straight from the rows' threads touch 32 lines
// each; while they drain, some 2500 cycles per tile, no barrier of the SM
// advances.)
//
// Only blocks with a visible key are loaded.  A page that ends inside a
// block is loaded as boxes of its own rows; boxes without a key, or whose keys
// no token of the sequence sees, are asked for outside the tensor, which TMA
// fills with zeros.
//
// Whole units (many of them) are dealt out in rounds, the longest rows first
// and every other round backwards.  Few units (STREAM, paged only) are cut:
// all units' blocks form one line, and every CTA takes an equal stretch of it,
// whatever the lengths of the sequences, which only the device knows (or an
// equal number of whole units, where that takes no longer).  A unit that lies
// in one stretch is finished by its CTA; of one that is cut, every CTA writes
// its part (O unnormalised, maximum, sum) to the workspace and the CTA that
// arrives last joins the parts in their order, at once: left to the end of
// the CTAs' work, the joins met there (16 chunks of 512 over 2K: 231 -> 249 us).
//
// What bounds it, bf16, D 128, 32 heads over 8 (B200, 6.55 TB/s and 1650
// TFLOP/s measured; under sustained load with inputs that change from pass to
// pass, in brackets a short loop over the same inputs, as are the figures
// beside the rules and steps below):
//   prefill of 8192, window 1024   173 us (151), 747 TFLOP/s of the visible
//                                  pairs; the tensor pipe and the exp2 unit are
//                                  both busy 53 % of the time: a step of a pair
//                                  of tiles (2.1 us) is the chain S -> maximum
//                                  -> exp2 -> P -> PV, twice, half overlapped
//   4 x 4096 causal                534 us, 1030 TFLOP/s, as above
//   64 single tokens, 0.8K..8K     218 us (192), 0.80 of the copy rate: HBM
//   2 single tokens, 4 kv heads,   101 us (97), 0.80 of it: HBM, and SMs that
//     128K                         end up to a quarter before the last
//   one token over 777             11.3 us (11.0): launch, a chain of dependent
//                                  loads (length, page, K, V) and the join
//   4 chunks of 512 over 8K        277 us (235), 865 TFLOP/s; as the prefill
#include <algorithm>

#include "attn_ops.cuh"

namespace gpo {

constexpr int kFwdMaxStages = 3;       // slots of the K ring and of the V ring
constexpr int kFwdSBufs = 3;           // S/P buffers (TILES = 1)
constexpr float kFwdRescale = 8.0f;    // see the softmax
constexpr int kFwdMaxCtas = 160;       // CTAs that a workspace has room for
// Blocks' time that writing and joining parts takes.  0, 2, 5, 12, window
// 1024: 4 chunks of 512 over 8K 83.4, 83.5, 59.2, 59.1 us; 12 chunks of up to
// 300 over 6K 31.7, 20.3, 20.2, 20.2.
constexpr int kFwdCutCost = 5;
constexpr int kFwdStreamPairs = 1024;  // most (sequence, span) pairs of a cut launch
// Registers of TILES = 2: 384 threads launch at 168; 128 * 88 + 256 * 208 is
// the same total (a softmax thread holds a row of 128 scores).
constexpr int kFwdLowRegs = 88, kFwdHighRegs = 208;
static_assert(128 * kFwdLowRegs + 256 * kFwdHighRegs <= 168 * 384,
              "register split exceeds the launch's registers");

// A stretch of a unit: blocks [i0, i1) of the n that its span sees.
struct FwdSeg {
  int b, h, t0, t1;  // tokens [t0, t1) of the span
  AttnSeq seq;
  AttnBlocks blk;
  int i0, i1;
  int64_t line0;  // cut launches: position of the unit's first block
  int unit;
  bool whole;
};

// Tile t of a stretch: its tokens and which of the span's blocks it sees.
struct FwdTile {
  int t0, t1, first, last, sinks;
  __device__ __forceinline__ bool sees(int block) const {
    return block <= last && (block >= first || block < sinks);
  }
};

// What warp 2 hands to the other roles (a single thread takes 3500 cycles to
// work a stretch out, which every role had to wait for when each did it).
struct FwdWork {
  FwdSeg seg;
  FwdTile tile[2];
  int more;  // 0: no stretch, the CTA is done
};

struct FwdShared {
  FwdWork work[2];
  uint64_t work_full[2], work_empty[2];

  uint64_t q_full, q_empty;
  uint64_t k_full[kFwdMaxStages], k_empty[kFwdMaxStages];
  uint64_t v_full[kFwdMaxStages], v_empty[kFwdMaxStages];
  uint64_t v_raw[kFwdMaxStages];  // copied, to be cleared before v_full (fwd_clears)
  uint64_t s_full[kFwdSBufs], p_full[kFwdSBufs], p_half[2], pv_done[kFwdSBufs];
  uint64_t o_full[2], o_free[2];
  // One staging tile for both tiles of O.  Use u has been stored when phase
  // u / 4 of stage_empty[u % 4] is done: a warpgroup without blocks can be two
  // units ahead of the other, more than one barrier's two phases can tell.
  uint64_t stage_full, stage_empty[4];
  int stage_at[8][3];                // batch, head, first row of the coming uses
  uint64_t drain;
  // cut launches: where this CTA's stretch begins
  int64_t line_pos, line_end, line_len;
  int64_t warp_sum[8];
  int warp_units[8], warp_longest[8];
  bool line_whole;  // positions count units, not blocks
  int line_pair, line_head, line_off;
  int last[2];
  uint32_t tmem_base;
  int abort;
};

struct FwdArgs {
  AttnGeom geom;
  void* out;
  float* lse;  // (batch, q_len, heads) or (tokens, heads); may be null
  int64_t o_batch, o_token, o_head;
  float scale_log2;
  int spans;     // units of a sequence and kv head (of the longest sequence)
  int items;
  int k_stages, v_stages;
  bool wide;     // rows of out on 32 bytes
  // cut launches
  unsigned int* arrived;  // per unit and tile, 0 between launches
  float* part;            // [CTA][2] parts of part_rows rows: D floats each, then (m, l)
  int part_rows;
  unsigned int* err;
};

struct RingPos2 {
  int slot = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void step(int stages) {
    if (++slot == stages) {
      slot = 0;
      parity ^= 1u;
    }
  }
};

// The CTA's stretches in order.
template <bool PAGED, bool STREAM, int TILES>
struct FwdWalk {
  const FwdArgs& a;
  FwdSeg s;
  int item, turn;     // whole units: first item of the CTA's turn
  int64_t pos, end;   // cut: positions in the line of blocks
  int pair, head, off, n, known;
  bool whole;

  __device__ __forceinline__ FwdWalk(const FwdArgs& args, const FwdShared& sh) : a(args) {
    item = 0;
    turn = 0;
    if constexpr (STREAM) {
      pos = sh.line_pos;
      end = sh.line_end;
      pair = sh.line_pair;
      head = sh.line_head;
      off = sh.line_off;
      whole = sh.line_whole;
      known = -1;
      n = 0;
    }
  }

  __device__ __forceinline__ void place(int r) {
    const AttnGeom& g = a.geom;
    s.b = r % g.batch;
    s.seq = attn_seq<PAGED>(g, s.b, a.err);
    s.t0 = (a.spans - 1 - r / g.batch) * TILES * g.tpt;  // the longest rows first
    s.t1 = min(s.t0 + TILES * g.tpt, s.seq.q_len);
    s.blk = attn_blocks(g, s.seq, s.t0, s.t1);
  }

  // The next stretch with a query (its rows may see no key: i0 == i1).
  __device__ __forceinline__ bool next() {
    const AttnGeom& g = a.geom;
    if constexpr (!STREAM) {
      // The longest units come first, and every other round runs backwards:
      // a CTA that had the longest of a round takes the shortest of the next.
      while (item < a.items) {
        const int mine = item + static_cast<int>((turn & 1) ? gridDim.x - 1 - blockIdx.x
                                                            : blockIdx.x);
        item += gridDim.x;
        ++turn;
        if (mine >= a.items) continue;
        s.h = mine % g.heads_kv;
        place(mine / g.heads_kv);
        if (s.t0 >= s.t1) continue;
        s.i0 = 0;
        s.i1 = s.blk.n;
        s.whole = true;
        return true;
      }
      return false;
    } else {
      if (pos >= end) return false;
      while (known != pair) {
        place(pair);
        known = pair;
        n = s.t0 < s.t1 ? max(1, s.blk.n) : 0;  // rows without a key: one empty block
        if (n == 0) ++pair;
      }
      s.h = head;
      s.unit = pair * g.heads_kv + head;
      s.line0 = pos - off;
      s.i0 = off;
      s.i1 = whole ? n : static_cast<int>(min(static_cast<int64_t>(n), off + (end - pos)));
      s.whole = s.i0 == 0 && s.i1 == n;
      pos += whole ? 1 : s.i1 - s.i0;
      off = s.i1;
      if (off == n) {
        off = 0;
        if (++head == g.heads_kv) {
          head = 0;
          ++pair;
        }
      }
      if (s.blk.n == 0) s.i1 = s.i0;
      return true;
    }
  }
};

__device__ __forceinline__ FwdTile fwd_tile(const AttnGeom& g, const FwdSeg& s, int t) {
  FwdTile f;
  f.t0 = s.t0 + t * g.tpt;
  f.t1 = min(f.t0 + g.tpt, s.seq.q_len);
  const AttnBlocks b = attn_blocks(g, s.seq, f.t0, f.t1);
  f.first = b.first;
  f.sinks = b.sink_blocks;
  f.last = b.n > 0 ? b.first + b.n - b.sink_blocks - 1 : -1;
  return f;
}

// Whether tile f of a stretch leaves through the staging tile: a whole
// unit's, of full height where the tensor would go on behind it.
template <bool PAGED, bool STREAM>
__device__ __forceinline__ bool fwd_staged(const AttnGeom& g, const FwdSeg& s, const FwdTile& f) {
  return f.t0 < f.t1 && (!STREAM || s.whole) && (!PAGED || f.t1 - f.t0 == g.tpt);
}

// Warp 2: works out the CTA's stretches, up to two ahead of their readers,
// and stores the staging tile whenever a warpgroup has filled it.
template <int D, bool PAGED, bool STREAM, int TILES>
__device__ __forceinline__ void fwd_schedule(const FwdArgs& args, FwdShared& sh,
                                             const CUtensorMap* tma_o, uint32_t stage) {
  FwdWalk<PAGED, STREAM, TILES> w(args, sh);
  bool more = true;
  uint32_t uses = 0, stored = 0;  // of the staging tile: planned, done
  unsigned long long idle_since = globaltimer_ns();
  for (uint32_t n = 0, poll = 1; more || stored < uses; ++poll) {
    bool moved = false;
    if (more && (n < 2 || mbar_test_wait(smem_u32(&sh.work_empty[n & 1]), ((n >> 1) - 1) & 1u))) {
      FwdWork& to = sh.work[n & 1];
      more = w.next();
      to.more = more ? 1 : 0;
      if (more) {
        to.seg = w.s;
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
          const FwdTile f = fwd_tile(args.geom, w.s, t);
          to.tile[t] = f;
          if (TILES == 2 && fwd_staged<PAGED, STREAM>(args.geom, w.s, f)) {
            int* at = sh.stage_at[uses & 7];
            at[0] = PAGED ? 0 : w.s.b;
            at[1] = w.s.h;
            at[2] = w.s.seq.row0 + f.t0;
            ++uses;
          }
        }
      }
      mbar_arrive(smem_u32(&sh.work_full[n & 1]));
      ++n;
      moved = true;
    }
    if (TILES == 2 && stored < uses && mbar_test_wait(smem_u32(&sh.stage_full), stored & 1u)) {
      const int* at = sh.stage_at[stored & 7];
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
        tma_store_5d(tma_o, stage + c * 128 * 128, c * 64, 0, at[1], at[2], at[0]);
      bulk_commit();
      bulk_wait_read();
      mbar_arrive(smem_u32(&sh.stage_empty[stored & 3]));
      ++stored;
      moved = true;
    }
    if (moved) {
      idle_since = globaltimer_ns();
    } else {
      __nanosleep(64);
      // The longest pause between two stretches is the work on one of them;
      // the roles at it have their own limit per wait and raise the flag.
      if ((poll & 255u) == 0 &&
          (*reinterpret_cast<volatile int*>(&sh.abort) ||
           globaltimer_ns() - idle_since > 16 * kWaitLimitNs)) {
        atomicOr(args.err, kErrWaitProducer);
        sh.abort = 1;
        break;
      }
    }
  }
  if (TILES == 2) bulk_wait();  // the last stores are out
}

// The n-th stretch for one role: false when there is none (or a wait failed).
template <bool WARP>
__device__ __forceinline__ bool fwd_take(FwdShared& sh, uint32_t& n, FwdSeg& s, unsigned int* err,
                                         uint32_t site, bool& ok) {
  const int i = n & 1u;
  ok = mbar_wait(smem_u32(&sh.work_full[i]), (n >> 1) & 1u, &sh.abort, err, site);
  if (WARP) ok = __all_sync(0xffffffffu, ok);
  if (!ok) return false;
  const bool more = *reinterpret_cast<volatile int*>(&sh.work[i].more) != 0;
  if (more) s = sh.work[i].seg;
  return more;
}
template <bool WARP>
__device__ __forceinline__ void fwd_taken(FwdShared& sh, uint32_t& n) {
  if (WARP) __syncwarp();
  if (!WARP || (threadIdx.x & 31) == 0) mbar_arrive(smem_u32(&sh.work_empty[n & 1u]));
  ++n;
}

// Cut launches: the blocks of every (sequence, span) pair are counted, and
// the pair where this CTA's stretch begins is found by a prefix sum.
template <bool PAGED, int TILES>
__device__ __forceinline__ void fwd_stretch(const FwdArgs& a, FwdShared& sh) {
  const AttnGeom& g = a.geom;
  const int pairs = a.spans * g.batch;
  const int per = (pairs + 255) / 256;
  const int tid = threadIdx.x, lane = tid & 31;
  FwdWalk<PAGED, false, TILES> w(a, sh);
  int cnt[kFwdStreamPairs / 256];
  // blocks, units (times heads) and the longest unit
  int64_t blocks = 0;
  int units = 0, longest = 0;
  if (tid < 256) {
#pragma unroll
    for (int i = 0; i < kFwdStreamPairs / 256; ++i) {
      cnt[i] = 0;
      const int r = tid * per + i;
      if (i < per && r < pairs) {
        w.place(r);
        cnt[i] = w.s.t0 < w.s.t1 ? max(1, w.s.blk.n) : 0;
        blocks += cnt[i];
        units += cnt[i] > 0 ? 1 : 0;
        longest = max(longest, cnt[i]);
      }
    }
  }
  int64_t incl = blocks;
  int incl_u = units;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
    const int up_u = __shfl_up_sync(0xffffffffu, incl_u, o);
    if (lane >= o) {
      incl += up;
      incl_u += up_u;
    }
    longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, o));
  }
  if (tid < 256 && lane == 31) {
    sh.warp_sum[tid >> 5] = incl;
    sh.warp_units[tid >> 5] = incl_u;
    sh.warp_longest[tid >> 5] = longest;
  }
  __syncthreads();
  int64_t before = incl - blocks, total = 0;
  int before_u = incl_u - units, total_u = 0;
  longest = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i < (tid >> 5)) {
      before += sh.warp_sum[i];
      before_u += sh.warp_units[i];
    }
    total += sh.warp_sum[i];
    total_u += sh.warp_units[i];
    longest = max(longest, sh.warp_longest[i]);
  }
  total *= g.heads_kv;
  const int64_t all_u = static_cast<int64_t>(total_u) * g.heads_kv;
  const int64_t ctas = gridDim.x;
  // Whole units where that takes no longer than cut ones and their joins.
  const bool whole = (all_u + ctas - 1) / ctas * longest <= (total + ctas - 1) / ctas + kFwdCutCost;
  if (whole) {
    before = before_u;
    total = all_u;
  }
  const int64_t len = (total + ctas - 1) / ctas;
  const int64_t p0 = min(total, len * blockIdx.x), p1 = min(total, p0 + len);
  if (tid == 0) {
    sh.line_pos = p0;
    sh.line_end = p1;
    sh.line_len = len;
    sh.line_whole = whole;
  }
  if (tid < 256) {
#pragma unroll
    for (int i = 0; i < kFwdStreamPairs / 256; ++i) {
      const int c = whole ? (cnt[i] > 0 ? 1 : 0) : cnt[i];
      const int64_t b0 = before * g.heads_kv, b1 = b0 + static_cast<int64_t>(c) * g.heads_kv;
      if (p0 < p1 && p0 >= b0 && p0 < b1) {
        sh.line_pair = tid * per + i;
        sh.line_head = static_cast<int>((p0 - b0) / c);
        sh.line_off = static_cast<int>((p0 - b0) % c);
      }
      before += c;
    }
  }
}

// Floats of a part: rows of O, then (m, l) of each row, on 16 bytes.
__host__ __device__ constexpr int64_t fwd_part_floats(int64_t rows, int d) {
  return rows * d + ((2 * rows + 3) & ~static_cast<int64_t>(3));
}

template <int N>
__device__ __forceinline__ void fwd_regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fwd_regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ void fwd_barrier(int id) {
  asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory");
}
// The same, and whether all four warps say so.  A warp that leaves its work
// (done, or a wait gave up) votes no once: a warp whose last wait ended in time
// is not left at the barrier for good by one whose wait did not.
__device__ __forceinline__ bool fwd_vote(int id, bool yes) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
      "bar.red.and.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(yes ? 1u : 0u), "r"(id)
      : "memory");
  return all != 0;
}

// Joins the parts [c0, c1] of a unit with few rows (16 at most), in their
// order and against a running maximum.  A thread has every nx-th vector of four
// dims of one row; those of P parts are loaded before the first is used, as
// the loop is bound by the latency of these loads (one token over 8K: 15.1 us,
// with 8 parts of two vectors 16.2; 16 parts of two spill).
template <typename LoadMl, typename Load, typename Finish>
__device__ __forceinline__ void fwd_join(int id, int rows, int vecs, int c0, int c1,
                                         LoadMl&& load_ml, Load&& load, Finish&& finish) {
  constexpr int P = 16;
  const int nx = 128 / rows, r = id % rows;
  if (id / rows >= nx) return;
  for (int x = id / rows; x < vecs; x += nx) {
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = -INFINITY, sum = 0.f;
#pragma unroll 1
    for (int c = c0; c <= c1; c += P) {
      float2 ml[P];
      float4 v[P];
#pragma unroll
      for (int i = 0; i < P; ++i) {
        ml[i] = make_float2(-INFINITY, 0.f);
        if (c + i <= c1) {
          ml[i] = load_ml(c + i, r);
          v[i] = load(c + i, r, x);
        }
      }
      float top = m;
#pragma unroll
      for (int i = 0; i < P; ++i) top = fmaxf(top, ml[i].y != 0.f ? ml[i].x : -INFINITY);
      const float a = m == top ? 1.f : ex2_approx(m - top);
      m = top;
      sum *= a;
      o.x *= a;
      o.y *= a;
      o.z *= a;
      o.w *= a;
#pragma unroll
      for (int i = 0; i < P; ++i)
        if (ml[i].y != 0.f) {  // a part without a key says nothing
          const float f = ex2_approx(ml[i].x - top);
          sum += ml[i].y * f;
          o.x += v[i].x * f;
          o.y += v[i].y * f;
          o.z += v[i].z * f;
          o.w += v[i].w * f;
        }
    }
    finish(r, x, o, m, sum);
  }
}

template <int D>
struct FwdGeom {
  static constexpr int SW = 128;  // swizzle atom: 64 dims of a row
  static constexpr int ATOMS = D / 64;
  static constexpr uint32_t Q_BYTES = 128u * D * 2;
  static constexpr uint32_t KV_BYTES = static_cast<uint32_t>(kOpsBN) * D * 2;
};

// Whether rows of a V block are cleared before the MMA reads it: slots behind
// a sequence's last key (paged; dense copies end there) and keys that no token
// sees hold anything.  P is 0 there, but 0 * NaN is not.  The copy of such a
// block ends at v_raw, and v_full is announced once it is cleared: the MMA
// thread, whose pace the others follow, has no part in it.  UNSEEN: the problem
// has keys that no token sees (paged: it may).
template <bool PAGED, bool UNSEEN>
__device__ __forceinline__ bool fwd_clears(const AttnGeom& g, const AttnSeq& s, int key0) {
  return (PAGED && key0 + kOpsBN > s.kv_len) ||
         (UNSEEN && key0 < attn_unseen(g, s) && attn_unseen_rows(g, s, key0).any());
}

// ---------------------------------------------------------------- producer
// K ring and Q (is_k), or V ring.  The whole warp runs the loop: each lane
// loads one box of a block.
template <int D, bool PAGED, bool UNSEEN, int TILES>
__device__ __forceinline__ void fwd_producer(const FwdArgs& args, FwdShared& sh,
                                             const CUtensorMap* tma_q, const CUtensorMap* map,
                                             uint32_t q_smem, uint32_t ring, bool is_k, int lane) {
  using G = FwdGeom<D>;
  const AttnGeom& g = args.geom;
  uint64_t* full = is_k ? sh.k_full : sh.v_full;
  uint64_t* empty = is_k ? sh.k_empty : sh.v_empty;
  volatile int* abort_flag = &sh.abort;
  const int boxes = PAGED ? kOpsBN / g.box_rows : 1;
  const int stages = is_k ? args.k_stages : args.v_stages;
  constexpr bool CLEARS = PAGED || UNSEEN;
  bool ok = true;
  int issued = 0, q_loads = 0;
  RingPos2 pos;
  uint32_t taken = 0;
  FwdSeg s;
  // The V block (its first key, -1: none) that is copied and not yet cleared.
  // It is cleared when the next slot of the ring is not free, so that the
  // blocks behind it are on their way meanwhile.
  int dirty = -1, dirty_slot = 0;
  uint32_t raw = 0, held = 0;  // bit s: parity of slot s's next v_raw phase; not cleared yet
  auto clear = [&]() {
    if (dirty < 0) return true;
    if (!__all_sync(0xffffffffu,
                    mbar_wait(smem_u32(&sh.v_raw[dirty_slot]), (raw >> dirty_slot) & 1u,
                              abort_flag, args.err, kErrWaitProducer)))
      return false;
    raw ^= 1u << dirty_slot;
    held &= ~(1u << dirty_slot);
    const uint32_t slot = ring + dirty_slot * G::KV_BYTES;
    constexpr int VECS = G::ATOMS * 8, ROWS = 32 / VECS;  // of a row; rows of a pass
    auto rows = [&](int r0, int r1) {
      for (int r = r0 + lane / VECS; r < r1; r += ROWS)
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                         slot + (lane % VECS / 8) * kOpsBN * G::SW + r * G::SW + (lane % 8) * 16),
                     "r"(0)
                     : "memory");
    };
    const AttnUnseenRows u = attn_unseen_rows(g, s.seq, dirty);
    rows(u.a0, u.a1);
    rows(u.b0, u.b1);
    if (PAGED) rows(s.seq.kv_len - dirty, kOpsBN);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&full[dirty_slot]));
    dirty = -1;
    return true;
  };
  while (fwd_take<true>(sh, taken, s, args.err, kErrWaitProducer, ok)) {
    fwd_taken<true>(sh, taken);
    if (s.i0 == s.i1) continue;
    if (is_k) {
      // Q of the previous stretch is free once its last S MMA is done
      ok = q_loads == 0 || mbar_wait(smem_u32(&sh.q_empty), (q_loads - 1) & 1u, abort_flag,
                                     args.err, kErrWaitProducer);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(smem_u32(&sh.q_full),
                              static_cast<uint32_t>(TILES * g.tpt * g.g) * D * 2);
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
          for (int c = 0; c < G::ATOMS; ++c)
            tma_load_5d(q_smem + t * G::Q_BYTES + c * 128 * G::SW, tma_q, smem_u32(&sh.q_full),
                        c * 64, 0, s.h, s.seq.row0 + s.t0 + t * g.tpt, PAGED ? 0 : s.b);
      }
      ++q_loads;
    }
    for (int i = s.i0; i < s.i1; ++i) {
      const int key0 = s.blk.at(i) * kOpsBN;
      int page = s.b, row = key0;
      if constexpr (PAGED) {
        const int key = key0 + lane * g.box_rows;
        // a page outside the tensor arrives as zeros (that of a cache without
        // pages has one all the same, as a tensor map cannot be empty)
        const int outside = max(g.num_pages, 1);
        page = outside;
        if (lane < boxes && key < s.seq.kv_len && !attn_box_unseen(g, s.seq, key)) {
          page = __ldg(g.table + s.b * g.table_stride + key / g.page_size);
          if (static_cast<unsigned int>(page) >= static_cast<unsigned int>(g.num_pages)) {
            page = outside;
            atomicOr(args.err, kErrBadLaunch);
          }
        }
        row = key % g.page_size;
      }
      const bool clears = !is_k && fwd_clears<PAGED, UNSEEN>(g, s.seq, key0);
      const uint32_t bar = smem_u32(clears ? &sh.v_raw[pos.slot] : &full[pos.slot]);
      const uint32_t free = smem_u32(&empty[pos.slot]);
      if (CLEARS && dirty >= 0 && !__all_sync(0xffffffffu, mbar_test_wait(free, pos.parity ^ 1u))) {
        ok = clear();
        if (!ok) break;
      }
      ok = __all_sync(0xffffffffu, mbar_wait(free, pos.parity ^ 1u, abort_flag, args.err,
                                             kErrWaitProducer));
      if (!ok) break;
      const uint32_t slot = ring + pos.slot * G::KV_BYTES;
      if (lane == 0) mbar_arrive_expect_tx(bar, G::KV_BYTES);
      __syncwarp();
      if (lane < boxes) {
        const uint32_t dst = slot + static_cast<uint32_t>(PAGED ? lane * g.box_rows : 0) * G::SW;
#pragma unroll
        for (int c = 0; c < G::ATOMS; ++c)
          tma_load_4d(dst + c * kOpsBN * G::SW, map, bar, c * 64, s.h, row, page);
      }
      ++issued;
      if (CLEARS && clears) {
        ok = clear();  // the one before
        dirty = key0;
        dirty_slot = pos.slot;
        held |= 1u << pos.slot;
        if (!ok) break;
      }
      pos.step(stages);
    }
    if (CLEARS && ok) ok = clear();
    if (!ok) break;
  }
  if (!ok && lane == 0) {
    // let the copies in flight land before the CTA can exit
    if (q_loads > 0) mbar_wait_drain(smem_u32(&sh.q_full), (q_loads - 1) & 1u, args.err);
    for (int j = max(0, issued - stages); j < issued; ++j) {
      const int at = j % stages;
      if (CLEARS && !is_k && ((held >> at) & 1u))
        mbar_wait_drain(smem_u32(&sh.v_raw[at]), (raw >> at) & 1u, args.err);
      else
        mbar_wait_drain(smem_u32(&full[at]), (j / stages) & 1u, args.err);
    }
  }
}

// -------------------------------------------------------------- MMA issuer
template <int FMT, int D, bool PAGED, int TILES>
__device__ __forceinline__ void fwd_mma(const FwdArgs& args, FwdShared& sh, uint32_t tmem,
                                        uint32_t q_smem, uint32_t k_smem, uint32_t v_smem) {
  using G = FwdGeom<D>;
  constexpr int BN = kOpsBN, SW = G::SW;
  constexpr uint32_t IDESC_S = make_idesc(FMT, 128, BN, false, false);
  constexpr uint32_t IDESC_O = make_idesc(FMT, 128, D, false, true);
  constexpr uint32_t S_COL = TILES * D;  // S/P buffers behind the O tiles
  constexpr uint64_t HI = smem_desc_hi(8 * SW, SW);
  unsigned int* err = args.err;
  volatile int* abort_flag = &sh.abort;
  // Between two MMA groups this thread does as little as it can: descriptor
  // halves advance by constants, waits test the phase without blocking first.
  auto wait = [&](const uint64_t* bar, uint32_t parity) {
    const uint32_t b = smem_u32(bar);
    return mbar_test_wait(b, parity) || mbar_wait(b, parity, abort_flag, err, kErrWaitMma);
  };
  const uint32_t q_lo = smem_desc_lo(q_smem, 16);
  const uint32_t k_lo = smem_desc_lo(k_smem, 16);
  const uint32_t v_lo = smem_desc_lo(v_smem, BN * SW);
  auto s_mma = [&](int t, int buf, int k_slot) {
    const uint32_t qd = q_lo + t * (G::Q_BYTES >> 4), kd = k_lo + k_slot * (G::KV_BYTES >> 4);
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      const uint32_t off = ((kk / 4) * 128 * SW + (kk % 4) * 32) >> 4;
      mma_f16_ss(tmem + S_COL + buf * BN, HI | (qd + off), HI | (kd + off), IDESC_S,
                 kk > 0 ? 1u : 0u);
    }
    mma_commit(smem_u32(&sh.s_full[buf]));
  };
  auto pv_part = [&](int t, int buf, int v_slot, int k0, int k1, bool first) {
    const uint32_t vd = v_lo + v_slot * (G::KV_BYTES >> 4);
    for (int kk = k0; kk < k1; ++kk)
      mma_f16_ts(tmem + t * D, tmem + S_COL + buf * BN + kk * 8,
                 HI | (vd + ((kk * 16 * SW) >> 4)), IDESC_O, (first && kk == 0) ? 0u : 1u);
  };
  bool ok = true;
  RingPos2 kpos, vpos;
  auto wait_v = [&]() { return wait(&sh.v_full[vpos.slot], vpos.parity); };
  uint32_t segs = 0, taken = 0;
  FwdSeg s;
  if constexpr (TILES == 1) {
    constexpr int NB = kFwdSBufs, LAG = NB - 1;
    RingPos2 spos, ppos;
    while (fwd_take<false>(sh, taken, s, err, kErrWaitMma, ok)) {
      fwd_taken<false>(sh, taken);
      const int n = s.i1 - s.i0;
      if (n == 0) continue;
      ok = wait(&sh.q_full, segs & 1u);
      for (int i = 0; i < n + LAG && ok; ++i) {
        if (i < n) {
          // S buffer i % NB last held P of block i - NB, whose PV MMA was
          // issued before; MMAs of one thread execute in issue order
          ok = wait(&sh.k_full[kpos.slot], kpos.parity);
          if (!ok) break;
          s_mma(0, spos.slot, kpos.slot);
          mma_commit(smem_u32(&sh.k_empty[kpos.slot]));
          if (i == n - 1) mma_commit(smem_u32(&sh.q_empty));
          kpos.step(args.k_stages);
          spos.step(NB);
        }
        const int j = i - LAG;
        if (j >= 0) {
          ok = wait_v() && wait(&sh.p_full[ppos.slot], ppos.parity);
          // the first PV overwrites O: the last epilogue has read it
          if (ok && j == 0 && segs > 0) ok = wait(&sh.o_free[0], (segs - 1) & 1u);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < BN / 16; kk += 4)
            pv_part(0, ppos.slot, vpos.slot, kk, kk + 4, j == 0);
          mma_commit(smem_u32(&sh.pv_done[ppos.slot]));
          mma_commit(smem_u32(&sh.v_empty[vpos.slot]));
          if (j == n - 1) mma_commit(smem_u32(&sh.o_full[0]));
          vpos.step(args.v_stages);
          ppos.step(NB);
        }
      }
      if (!ok) break;
      ++segs;
    }
  } else {
    uint32_t blocks[2] = {0u, 0u};  // blocks of each tile so far: phases of its P
    uint32_t outs[2] = {0u, 0u};    // stretches in which the tile had a block
    while (fwd_take<false>(sh, taken, s, err, kErrWaitMma, ok)) {
      const FwdTile tile[2] = {sh.work[taken & 1u].tile[0], sh.work[taken & 1u].tile[1]};
      fwd_taken<false>(sh, taken);
      if (s.i0 == s.i1) continue;
      auto sees = [&](int t, int i) { return tile[t].sees(s.blk.at(i)); };
      bool begun[2] = {false, false};
      ok = wait(&sh.q_full, segs & 1u) && wait(&sh.k_full[kpos.slot], kpos.parity);
      if (!ok) break;
      // S_t of a stretch's first block overwrites the P that the last PV_t of
      // the stretch before read: it was issued before, MMAs run in order
      bool now[2], then[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        now[t] = sees(t, s.i0);
        if (now[t]) s_mma(t, t, kpos.slot);
      }
      mma_commit(smem_u32(&sh.k_empty[kpos.slot]));
      kpos.step(args.k_stages);
      if (s.i1 - s.i0 == 1) mma_commit(smem_u32(&sh.q_empty));
      for (int i = s.i0; i < s.i1; ++i) {
        const bool more = i + 1 < s.i1;
#pragma unroll
        for (int t = 0; t < 2; ++t) then[t] = more && sees(t, i + 1);
        ok = wait_v();
        if (!ok) break;
        bool k_ready = false;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (now[t]) {
            // a tile's first PV overwrites O_t: the last epilogue has read it
            if (!begun[t] && outs[t] > 0) ok = wait(&sh.o_free[t], (outs[t] - 1) & 1u);
            if (!ok) break;
            // keys [0, 64) as soon as their P is stored, then the rest
            const uint32_t par = blocks[t] & 1u;
            const bool all = mbar_test_wait(smem_u32(&sh.p_full[t]), par);
            if (!all) {
              ok = wait(&sh.p_half[t], par);
              if (!ok) break;
            }
            tc_fence_after();
#pragma unroll
            for (int kk = 0; kk < BN / 32; ++kk)
              pv_part(t, t, vpos.slot, kk, kk + 1, !begun[t]);
            if (!all) {
              ok = wait(&sh.p_full[t], par);
              if (!ok) break;
              tc_fence_after();
            }
#pragma unroll
            for (int kk = BN / 32; kk < BN / 16; ++kk)
              pv_part(t, t, vpos.slot, kk, kk + 1, false);
            begun[t] = true;
            ++blocks[t];
            if (!then[t]) {
              // the tile's last block, unless it skips some (a gap between
              // its sinks and its window that the other tile sees)
              bool end = true;
              for (int x = i + 2; x < s.i1 && end; ++x) end = !sees(t, x);
              if (end) {
                mma_commit(smem_u32(&sh.o_full[t]));
                ++outs[t];
              }
            }
          }
          if (then[t]) {
            if (!k_ready) {
              ok = wait(&sh.k_full[kpos.slot], kpos.parity);
              if (!ok) break;
              k_ready = true;
            }
            s_mma(t, t, kpos.slot);
          }
        }
        if (ok && more && !k_ready) ok = wait(&sh.k_full[kpos.slot], kpos.parity);
        if (!ok) break;
        if (more) {
          mma_commit(smem_u32(&sh.k_empty[kpos.slot]));
          if (i + 2 == s.i1) mma_commit(smem_u32(&sh.q_empty));
          kpos.step(args.k_stages);
        }
        mma_commit(smem_u32(&sh.v_empty[vpos.slot]));
        vpos.step(args.v_stages);
#pragma unroll
        for (int t = 0; t < 2; ++t) now[t] = then[t];
      }
      if (!ok) break;
      ++segs;
    }
  }
  if (!ok) {
    mma_commit(smem_u32(&sh.drain));
    mbar_wait_drain(smem_u32(&sh.drain), 0, err);
  }
}

// ---------------------------------------------------- softmax and epilogue
template <typename T, int FMT, int D, bool PAGED, bool STREAM, int TILES>
__device__ __forceinline__ void fwd_softmax(const FwdArgs& args, FwdShared& sh, uint32_t stage,
                                            uint32_t tmem, int warp, int lane) {
  constexpr int BN = kOpsBN;
  constexpr uint32_t S_COL = TILES * D;
  const AttnGeom& g = args.geom;
  unsigned int* err = args.err;
  volatile int* abort_flag = &sh.abort;
  const int t = TILES == 1 ? 0 : (warp - 4) >> 2;
  const int q = warp & 3;
  const int row = q * 32 + lane;
  const uint32_t lane_addr = static_cast<uint32_t>(q * 32) << 16;
  const uint32_t o_tmem = tmem + lane_addr + t * D;
  const float2 scale2 = make_float2(args.scale_log2, args.scale_log2);
  const int row_token = row / g.g, row_head = row % g.g;
  auto wait = [&](const uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu,
                      mbar_wait(smem_u32(bar), parity, abort_flag, err, kErrWaitSoftmax));
  };
  bool ok = true;
  RingPos2 spos, last_pv;     // TILES = 1: S buffers
  uint32_t blocks = 0, outs = 0;
  uint32_t uses = 0;  // of the staging tile, by either tile
  if (TILES == 2) spos.slot = t;
  uint32_t taken = 0;
  FwdSeg s;
  while (fwd_take<true>(sh, taken, s, err, kErrWaitSoftmax, ok)) {
    const FwdTile tile = sh.work[taken & 1u].tile[t];
    // tile 0's use of the staging tile comes before tile 1's
    bool staged = false;
    uint32_t use = 0;
    if (TILES == 2) {
      const bool s0 = fwd_staged<PAGED, STREAM>(g, s, sh.work[taken & 1u].tile[0]);
      const bool s1 = fwd_staged<PAGED, STREAM>(g, s, sh.work[taken & 1u].tile[1]);
      staged = t == 0 ? s0 : s1;
      use = uses + (t == 1 && s0 ? 1u : 0u);
      uses += (s0 ? 1u : 0u) + (s1 ? 1u : 0u);
    }
    fwd_taken<true>(sh, taken);
    if (tile.t0 >= tile.t1) continue;
    const int token = tile.t0 + row_token;
    const bool live = row_token < g.tpt && token < tile.t1;
    const bool idle = q * 32 >= (tile.t1 - tile.t0) * g.g;  // no query in this warp
    const int p = token + s.seq.off;
    float m_used = -INFINITY, l = 0.f;
    int seen = 0;
    for (int i = s.i0; i < s.i1; ++i) {
      if (TILES == 2 && !tile.sees(s.blk.at(i))) continue;
      if (TILES == 2) spos.parity = blocks & 1u;
      ok = wait(&sh.s_full[spos.slot], spos.parity);
      if (!ok) break;
      if (idle) {
        // whatever the P rows of this warp hold reaches only its O rows
        __syncwarp();
        if (lane == 0) {
          if (TILES == 2) mbar_arrive(smem_u32(&sh.p_half[t]));
          mbar_arrive(smem_u32(&sh.p_full[spos.slot]));
        }
      } else {
        tc_fence_after();
        const uint32_t sp = tmem + lane_addr + S_COL + spos.slot * BN;
        uint32_t sv[BN];
#pragma unroll
        for (int c = 0; c < BN / 32; ++c)
          tmem_ld32(sp + c * 32, *reinterpret_cast<uint32_t(*)[32]>(sv + c * 32));
        tmem_wait_ld();
        auto f = [&](int e) { return __uint_as_float(sv[e]); };
        const int key0 = s.blk.at(i) * BN;
        if (block_is_masked(g, s.seq, tile.t0, tile.t1, key0)) {
          const RowMask rm = row_mask(g, p, key0);
#pragma unroll
          for (int c = 0; c < BN / 32; ++c) {
            const uint32_t see = rm.word(c);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              sv[c * 32 + e] = (see & (1u << e)) ? sv[c * 32 + e] : __float_as_uint(-INFINITY);
          }
        }
        float mx[4] = {f(0), f(1), f(2), f(3)};
#pragma unroll
        for (int e = 4; e + 1 < BN; e += 2)
          mx[(e >> 1) & 3] = fmax3(mx[(e >> 1) & 3], f(e), f(e + 1));
        const float mb = fmaxf(fmax3(mx[0], mx[1], mx[2]), mx[3]) * args.scale_log2;
        // The maximum that P is taken against moves only when a block's
        // exceeds it by 2^8 (or there is none yet): P <= 256 is as exact in
        // 16 bits as P <= 1, and O is rescaled in TMEM that rarely.
        if (seen == 0) {
          m_used = mb;
        } else {
          const bool need = mb > m_used + kFwdRescale;
          if (__any_sync(0xffffffffu, need)) {
            if (TILES == 1) {
              // O holds the PV of every earlier block once the last is done
              // (TILES = 2: S_t is issued behind the tile's last PV)
              ok = wait(&sh.pv_done[last_pv.slot], last_pv.parity);
              if (!ok) break;
              tc_fence_after();
            }
            const float m_new = need ? mb : m_used;
            const float alpha = need ? ex2_approx(m_used - m_new) : 1.f;
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t r[16];
              tmem_ld16(o_tmem + c * 16, r);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * alpha);
              tmem_st16(o_tmem + c * 16, r);
            }
            tmem_wait_st();
            l *= alpha;
            m_used = m_new;
          }
        }
        // a row that has seen nothing yet: -inf - 0, so that P is 0
        const float neg_m = (m_used == -INFINITY) ? 0.f : -m_used;
        const float2 shift2 = make_float2(neg_m, neg_m);
        float2 rs[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f),
                        make_float2(0.f, 0.f)};
        auto release = [&](uint64_t* bar) {
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(bar));
        };
#pragma unroll
        for (int c = 0; c < BN / 32; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int g2 = 0; g2 < 16; ++g2) {
            const int e = c * 16 + g2;
            const float2 x = __ffma2_rn(make_float2(f(2 * e), f(2 * e + 1)), scale2, shift2);
            const float2 pp = make_float2(ex2_approx(x.x), ex2_approx(x.y));  // -inf -> 0
            rs[e & 3] = __fadd2_rn(rs[e & 3], pp);
            // P in the inputs' type: the MMA takes both operands in one type
            pk[g2] = FMT == 1 ? pack_bf16(pp.x, pp.y) : pack_f16(pp.x, pp.y);
          }
          tmem_st16(sp + c * 16, pk);
          if (TILES == 2 && c == 1) release(&sh.p_half[t]);
        }
        release(&sh.p_full[spos.slot]);
        const float2 rsum = __fadd2_rn(__fadd2_rn(rs[0], rs[1]), __fadd2_rn(rs[2], rs[3]));
        l += rsum.x + rsum.y;
      }
      ++seen;
      if (TILES == 1) {
        last_pv = spos;
        spos.step(kFwdSBufs);
      } else {
        ++blocks;
      }
    }
    if (!ok) break;
    // ------------------------------------------------------------ epilogue
    uint32_t ov[D];
    if (seen > 0) {
      ok = wait(&sh.o_full[t], outs & 1u);
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < D / 32; ++c)
        tmem_ld32(o_tmem + c * 32, *reinterpret_cast<uint32_t(*)[32]>(ov + c * 32));
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.o_free[t]));
      ++outs;
    } else {
#pragma unroll
      for (int e = 0; e < D; ++e) ov[e] = 0u;
    }
    const int head = s.h * g.g + row_head;
    auto lse_at = [&](int64_t r, int tok, int hd) {
      return (PAGED ? r : static_cast<int64_t>(s.b) * g.q_len + tok) *
                 (static_cast<int64_t>(g.heads_kv) * g.g) + hd;
    };
    if (!STREAM || s.whole) {
      if (live && args.lse)
        args.lse[lse_at(s.seq.row0 + token, token, head)] =
            l == 0.f ? -INFINITY : (m_used + log2f(l)) * 0.6931471805599453f;
      const float inv_l = l == 0.f ? 0.f : 1.0f / l;
      T* orow = static_cast<T*>(args.out) + (PAGED ? 0 : s.b * args.o_batch) +
                (s.seq.row0 + token) * args.o_token + head * args.o_head;
      // the tile's last contents have been read out
      if (staged && use > 0) {
        ok = wait(&sh.stage_empty[(use - 1) & 3], ((use - 1) >> 2) & 1u);
        if (!ok) break;
      }
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        uint32_t pk[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float lo = __uint_as_float(ov[c * 16 + 2 * e]) * inv_l;
          const float hi = __uint_as_float(ov[c * 16 + 2 * e + 1]) * inv_l;
          pk[e] = FMT == 1 ? pack_bf16(lo, hi) : pack_f16(lo, hi);
        }
        if (staged) {
          stage_chunk(stage, row, 2 * c, pk);
          stage_chunk(stage, row, 2 * c + 1, pk + 4);
        } else if (live) {
          store_pairs8(orow + c * 16, pk, args.wide);
        }
      }
      if (staged) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.stage_full));
      }
      continue;
    }
    if constexpr (STREAM) {
      // ------------------------------------------------- parts of a cut unit
      const int64_t part_floats = fwd_part_floats(args.part_rows, D);
      const int c_first = static_cast<int>(s.line0 / sh.line_len);
      const int c_last = static_cast<int>((s.line0 + s.blk.n - 1) / sh.line_len);
      // a CTA has two parts at most: slot 0 of a unit that began before its
      // stretch, slot 1 of one that goes on behind it
      auto part_of = [&](int c) {
        return args.part + (2 * static_cast<int64_t>(c) + (c == c_first ? 1 : 0)) * part_floats;
      };
      auto part_ml = [&](float* part) {
        return reinterpret_cast<float2*>(part + static_cast<int64_t>(args.part_rows) * D);
      };
      const int base = t * g.tpt * g.g;  // this tile's rows in a part
      const int rows = (tile.t1 - tile.t0) * g.g;
      {
        // four dims of all rows, then the next four: a warp's stores and the
        // join's loads are contiguous
        float* mine = part_of(static_cast<int>(blockIdx.x));
        if (live) {
          float4* o4 = reinterpret_cast<float4*>(mine) + base + row;
          if (seen > 0)
#pragma unroll
            for (int c = 0; c < D / 4; ++c)
              __stcg(o4 + c * args.part_rows,
                     make_float4(__uint_as_float(ov[4 * c]), __uint_as_float(ov[4 * c + 1]),
                                 __uint_as_float(ov[4 * c + 2]), __uint_as_float(ov[4 * c + 3])));
          __stcg(part_ml(mine) + base + row, make_float2(m_used, l));
        }
      }
      __threadfence();
      if (!fwd_vote(1 + t, true)) return;
      if (row == 0) {
        unsigned int* cnt = args.arrived + static_cast<int64_t>(s.unit) * TILES + t;
        const unsigned int before = atomicAdd(cnt, 1u);
        const bool last = before == static_cast<unsigned int>(c_last - c_first);
        if (last) atomicExch(cnt, 0u);  // ready for the next launch
        sh.last[t] = last ? 1 : 0;
      }
      fwd_barrier(1 + t);
      const bool join = *reinterpret_cast<volatile int*>(&sh.last[t]) != 0;
      if (join) {
        __threadfence();
        // An element is four dims of a row.  Few rows come with many parts
        // (their unit spans many CTAs), many rows with two or three.
        auto finish = [&](int r, int x, const float4& o, float m, float sum) {
          const float inv = sum == 0.f ? 0.f : 1.0f / sum;
          const int tok = tile.t0 + r / g.g, hd = s.h * g.g + r % g.g;
          const int64_t at = s.seq.row0 + tok;
          if (args.lse && x == 0)
            args.lse[lse_at(at, tok, hd)] =
                sum == 0.f ? -INFINITY : (m + log2f(sum)) * 0.6931471805599453f;
          T* orow = static_cast<T*>(args.out) + at * args.o_token + hd * args.o_head;
          const uint32_t lo = FMT == 1 ? pack_bf16(o.x * inv, o.y * inv)
                                       : pack_f16(o.x * inv, o.y * inv);
          const uint32_t hi = FMT == 1 ? pack_bf16(o.z * inv, o.w * inv)
                                       : pack_f16(o.z * inv, o.w * inv);
          reinterpret_cast<uint2*>(orow)[x] = make_uint2(lo, hi);
        };
        auto load_ml = [&](int c, int r) { return __ldcg(part_ml(part_of(c)) + base + r); };
        auto load = [&](int c, int r, int x) {
          return __ldcg(reinterpret_cast<const float4*>(part_of(c)) + base + r +
                        x * args.part_rows);
        };
        // With two tiles the join of few rows spilled (4 chunks of 512 over 8K
        // 235 -> 270..350 us): rows each take a thread there.  Units of two
        // tiles have many rows and two or three parts, unless a plan that takes
        // chunks is called for single tokens (see fwd_tiles).
        if (TILES == 1 && rows <= 16) {
          if constexpr (TILES == 1)
            fwd_join(row, rows, D / 4, c_first, c_last, load_ml, load, finish);
        } else if (row < rows) {
          // thread = row: its weights first, then 32 dims of two parts at a
          // time (16 loads in flight), which leave as 32-byte stores
          float m = -INFINITY, sum = 0.f;
#pragma unroll 4
          for (int c = c_first; c <= c_last; ++c) {
            const float2 ml = __ldcg(part_ml(part_of(c)) + base + row);
            if (ml.y != 0.f) {
              const float to = fmaxf(m, ml.x);
              sum = sum * ex2_approx(m - to) + ml.y * ex2_approx(ml.x - to);
              m = to;
            }
          }
          const float inv = sum == 0.f ? 0.f : 1.0f / sum;
          const int64_t at = s.seq.row0 + token;
          if (args.lse)
            args.lse[lse_at(at, token, head)] =
                sum == 0.f ? -INFINITY : (m + log2f(sum)) * 0.6931471805599453f;
          T* orow = static_cast<T*>(args.out) + at * args.o_token + head * args.o_head;
#pragma unroll 1
          for (int x0 = 0; x0 < D / 4; x0 += 8) {
            float4 o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
            for (int c = c_first; c <= c_last; ++c) {
              float* part = part_of(c);
              const float2 ml = __ldcg(part_ml(part) + base + row);
              float4 v[8];
#pragma unroll
              for (int i = 0; i < 8; ++i)
                v[i] = __ldcg(reinterpret_cast<const float4*>(part) + base + row +
                              (x0 + i) * args.part_rows);
              if (ml.y != 0.f) {  // a part without a key says nothing
                const float f = ex2_approx(ml.x - m) * inv;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  o[i].x += v[i].x * f;
                  o[i].y += v[i].y * f;
                  o[i].z += v[i].z * f;
                  o[i].w += v[i].w * f;
                }
              }
            }
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              pk[2 * i] = FMT == 1 ? pack_bf16(o[i].x, o[i].y) : pack_f16(o[i].x, o[i].y);
              pk[2 * i + 1] = FMT == 1 ? pack_bf16(o[i].z, o[i].w) : pack_f16(o[i].z, o[i].w);
            }
            store_pairs8(orow + x0 * 4, pk, args.wide);
            store_pairs8(orow + x0 * 4 + 16, pk + 8, args.wide);
          }
        }
      }
    }
  }
  if (STREAM) fwd_vote(1 + t, false);
}

template <typename T, int FMT, int D, bool PAGED, bool STREAM, int TILES, bool UNSEEN>
__global__ void __launch_bounds__(128 + 128 * TILES, 1)
    attn_fwd_kernel(const __grid_constant__ CUtensorMap tma_q,
                    const __grid_constant__ CUtensorMap tma_k,
                    const __grid_constant__ CUtensorMap tma_v,
                    const __grid_constant__ CUtensorMap tma_o,
                    const __grid_constant__ FwdArgs args) {
  using G = FwdGeom<D>;
  constexpr int NB = TILES == 1 ? kFwdSBufs : 2;
  static_assert(TILES * D + NB * kOpsBN <= 512, "TMEM holds 512 columns");

  __shared__ FwdShared sh;
  extern __shared__ uint8_t dyn_smem[];
  const uint32_t base = (smem_u32(dyn_smem) + 1023u) & ~1023u;
  const uint32_t q_smem = base;
  const uint32_t k_smem = q_smem + TILES * G::Q_BYTES;
  const uint32_t v_smem = k_smem + args.k_stages * G::KV_BYTES;
  const uint32_t stage = v_smem + args.v_stages * G::KV_BYTES;  // TILES = 2
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&sh.q_full), 1);
    mbar_init(smem_u32(&sh.q_empty), 1);
    for (int s = 0; s < kFwdMaxStages; ++s) {
      mbar_init(smem_u32(&sh.k_full[s]), 1);
      mbar_init(smem_u32(&sh.k_empty[s]), 1);
      mbar_init(smem_u32(&sh.v_full[s]), 1);
      mbar_init(smem_u32(&sh.v_empty[s]), 1);
      mbar_init(smem_u32(&sh.v_raw[s]), 1);
    }
    for (int b = 0; b < NB; ++b) {
      mbar_init(smem_u32(&sh.s_full[b]), 1);
      mbar_init(smem_u32(&sh.p_full[b]), 4);
      mbar_init(smem_u32(&sh.pv_done[b]), 1);
    }
    for (int t = 0; t < TILES; ++t) {
      mbar_init(smem_u32(&sh.p_half[t]), 4);
      mbar_init(smem_u32(&sh.o_full[t]), 1);
      mbar_init(smem_u32(&sh.o_free[t]), 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&sh.work_full[i]), 1);
      mbar_init(smem_u32(&sh.work_empty[i]), 3 + 4 * TILES);  // two producers, MMA, softmax warps
    }
    mbar_init(smem_u32(&sh.stage_full), 4);
    for (int i = 0; i < 4; ++i) mbar_init(smem_u32(&sh.stage_empty[i]), 1);
    mbar_init(smem_u32(&sh.drain), 1);
    sh.abort = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tma_q);
    tma_prefetch_desc(&tma_k);
    tma_prefetch_desc(&tma_v);
    if (TILES == 2) tma_prefetch_desc(&tma_o);
  }
  if (warp == 2) {
    tmem_alloc(smem_u32(&sh.tmem_base), 512);
    tmem_relinquish();
  }
  let_next_start();
  if constexpr (STREAM) {
    wait_for_previous();
    fwd_stretch<PAGED, TILES>(args, sh);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem_base;
  if constexpr (!STREAM) wait_for_previous();

  if (warp < 4) {
    if constexpr (TILES == 2) fwd_regs_dec<kFwdLowRegs>();
    if (warp == 0 || warp == 3)
      fwd_producer<D, PAGED, UNSEEN, TILES>(args, sh, &tma_q, warp == 0 ? &tma_k : &tma_v, q_smem,
                                    warp == 0 ? k_smem : v_smem, warp == 0, lane);
    else if (warp == 1 && elect_one())
      fwd_mma<FMT, D, PAGED, TILES>(args, sh, tmem, q_smem, k_smem, v_smem);
    else if (warp == 2 && elect_one())
      fwd_schedule<D, PAGED, STREAM, TILES>(args, sh, &tma_o, stage);
  } else {
    if constexpr (TILES == 2) fwd_regs_inc<kFwdHighRegs>();
    fwd_softmax<T, FMT, D, PAGED, STREAM, TILES>(args, sh, stage, tmem, warp, lane);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2) tmem_dealloc(tmem, 512);
}

// ------------------------------------------------------------------- host
typedef CUresult (*OpsEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static bool encode_ops_map(CUtensorMap* map, int dtype, const void* ptr, int rank,
                           const cuuint64_t* dims, const int64_t* strides,
                           const cuuint32_t* box) {
  OpsEncodeFn fn = reinterpret_cast<OpsEncodeFn>(tensor_map_encoder());
  if (!fn) return false;
  cuuint64_t bytes[4];
  // a dimension of one element is never stepped over: any valid stride does
  for (int i = 0; i + 1 < rank; ++i)
    bytes[i] = dims[i + 1] == 1 ? 16u : static_cast<cuuint64_t>(strides[i]) * 2u;
  const cuuint32_t step[5] = {1, 1, 1, 1, 1};
  return fn(map,
            dtype == GPO_BFLOAT16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                  : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
            static_cast<cuuint32_t>(rank), const_cast<void*>(ptr), dims, bytes, box, step,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool encode_rows_map(CUtensorMap* map, int dtype, const HeadsView& t, int dim, int g, int tpt) {
  const cuuint64_t dims[5] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(g),
                              static_cast<cuuint64_t>(t.heads / g),
                              static_cast<cuuint64_t>(t.tokens), static_cast<cuuint64_t>(t.batch)};
  const int64_t strides[4] = {t.s_head, t.s_head * g, t.s_token, t.s_batch};
  const cuuint32_t box[5] = {64, static_cast<cuuint32_t>(g), 1, static_cast<cuuint32_t>(tpt), 1};
  return encode_ops_map(map, dtype, t.ptr, 5, dims, strides, box);
}

bool encode_keys_map(CUtensorMap* map, int dtype, const HeadsView& t, int dim, int rows) {
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(t.heads),
                              static_cast<cuuint64_t>(t.tokens), static_cast<cuuint64_t>(t.batch)};
  const int64_t strides[3] = {t.s_head, t.s_token, t.s_batch};
  const cuuint32_t box[4] = {64, 1, static_cast<cuuint32_t>(rows), 1};
  return encode_ops_map(map, dtype, t.ptr, 4, dims, strides, box);
}

namespace {

// Two tiles per unit where a sequence fills them and where every SM gets
// more than two tiles: with fewer, a tile per CTA ends earlier.  One tile
// against two, bf16, D 128, 32 heads over 8, window 1024: 1 x 512 tokens
// 10.6 / 14.4 us, 1024 17.3 / 22.6, 2048 43.5 / 41.5, 8192 183 / 155; paged,
// 4 chunks of 512 over 8K 293 / 247.  The host knows max_q, not the lengths: a
// call for single tokens from a plan that takes chunks gets two tiles, one of
// them empty (64 tokens over 0.8K..8K from a plan of max_q 1 / 512: 196 / 252
// us; with a window of 1024 65 / 91; 256 over 0.2K..2K 238 / 317; 16 tokens 52
// / 52).  A plan for each kind of step avoids it.
int fwd_tiles(const AttnGeom& g) {
  int64_t tiles = static_cast<int64_t>(cdiv(g.q_len, g.tpt)) * g.batch;
  // paged: the rows of all sequences together fill no more than
  if (g.kv_lens) tiles = std::min<int64_t>(tiles, g.tokens / g.tpt + g.batch);
  return g.q_len > g.tpt && tiles * g.heads_kv > 2 * kFwdMaxCtas ? 2 : 1;
}

int fwd_spans(const AttnGeom& g) {
  return static_cast<int>(cdiv(static_cast<uint64_t>(g.q_len),
                               static_cast<uint64_t>(fwd_tiles(g)) * g.tpt));
}

// Units are cut where whole ones would leave SMs idle in the last round:
// fewer than eight rounds of them.  Cut against whole (us): single tokens
// over 2 x 128K 98 / 1097, over 64 x 0.8K..8K 191 / 232; chunks of up to 300
// over 12 x 1.2K..6K, window 1024, 20.2 / 40.2; 4 chunks of 512 over 8K
// 231 / 237.  Where lengths happen to fill the rounds, whole units would win
// (single tokens over 128 x 2K 116 / 109, 16 chunks of 512 over 2K 236 / 206),
// but the lengths are on the device: cutting lost 15 % at most, whole units
// lose any factor.
bool fwd_is_cut(const AttnGeom& g) {
  const int64_t pairs = static_cast<int64_t>(fwd_spans(g)) * g.batch;
  return pairs <= kFwdStreamPairs && pairs * g.heads_kv < 8 * kFwdMaxCtas;
}

int fwd_part_rows(const AttnGeom& g) {
  return std::min(fwd_tiles(g) * g.tpt, g.q_len) * g.g;
}

// Counters come first and have a fixed size, so that calls of one plan with
// different batches agree on where they are (and that they are zero).
uint64_t fwd_counter_bytes(const AttnGeom& g) {
  return (static_cast<uint64_t>(8 * kFwdMaxCtas) + g.heads_kv) * 2u * sizeof(unsigned int);
}

template <typename T, int FMT, int D, bool PAGED, bool STREAM, int TILES, bool UNSEEN = PAGED>
gpo_status run_fwd(const AttnProblem& p, const LaunchCtx& c) {
  const AttnGeom& g = p.geom;
  CUtensorMap mq, mk, mv, mo;
  const HeadsView out{p.out, p.q.batch, p.q.tokens, p.q.heads, p.o_batch, p.o_token, p.o_head};
  if (!encode_rows_map(&mq, p.dtype, p.q, D, g.g, g.tpt) ||
      !encode_rows_map(&mo, p.dtype, out, D, g.g, g.tpt) ||
      !encode_keys_map(&mk, p.dtype, p.k, D, g.box_rows) ||
      !encode_keys_map(&mv, p.dtype, p.v, D, g.box_rows))
    return GPO_BAD_ARGS;
  FwdArgs a{};
  a.geom = g;
  a.out = p.out;
  a.lse = p.lse;
  a.o_batch = p.o_batch;
  a.o_token = p.o_token;
  a.o_head = p.o_head;
  a.scale_log2 = p.scale * 1.4426950408889634f;
  a.spans = fwd_spans(g);
  // Two Q tiles and the staging tile of D = 128 leave room for four slots
  // (a third V slot in the staging tile's place measured the same).
  constexpr int STAGES = TILES == 1 || D == 64 ? kFwdMaxStages : 2;
  a.k_stages = a.v_stages = STAGES;
  a.wide = (reinterpret_cast<uintptr_t>(p.out) & 31u) == 0 && p.o_batch % 16 == 0 &&
           p.o_token % 16 == 0 && p.o_head % 16 == 0;
  a.err = c.err;
  const int64_t items = static_cast<int64_t>(a.spans) * g.batch * g.heads_kv;
  if (items > (1ll << 31) - 1024) return GPO_BAD_ARGS;
  a.items = static_cast<int>(items);
  const int sms = std::min(c.sm_count > 0 ? c.sm_count : 148, kFwdMaxCtas);
  int64_t ctas = std::min<int64_t>(items, sms);
  if (STREAM) {
    a.arrived = static_cast<unsigned int*>(p.workspace);
    a.part = reinterpret_cast<float*>(static_cast<char*>(p.workspace) +
                                      ((fwd_counter_bytes(g) + 255u) & ~255ull));
    a.part_rows = fwd_part_rows(g);
    ctas = sms;
  }
  auto kern = attn_fwd_kernel<T, FMT, D, PAGED, STREAM, TILES, UNSEEN>;
  constexpr uint32_t dyn =
      (TILES * 128u + 2u * STAGES * kOpsBN + (TILES == 2 ? 128u : 0u)) * D * 2u + 1024u;
  static_assert(dyn + sizeof(FwdShared) > kOpsAloneBytes, "two CTAs fit an SM");
  gpo_status s = ensure_smem_attr(reinterpret_cast<const void*>(kern), dyn);
  if (s != GPO_OK) return s;
  return launch_in_order(kern, static_cast<unsigned>(ctas), 128 + 128 * TILES, dyn, c.stream, mq,
                         mk, mv, mo, a);
}

template <typename T, int FMT, int D>
gpo_status run_fwd_form(const AttnProblem& p, const LaunchCtx& c) {
  const bool two = fwd_tiles(p.geom) == 2;
  if (!p.paged && attn_has_unseen(p.geom))
    return two ? run_fwd<T, FMT, D, false, false, 2, true>(p, c)
               : run_fwd<T, FMT, D, false, false, 1, true>(p, c);
  if (!p.paged)
    return two ? run_fwd<T, FMT, D, false, false, 2>(p, c)
               : run_fwd<T, FMT, D, false, false, 1>(p, c);
  if (fwd_is_cut(p.geom))
    return two ? run_fwd<T, FMT, D, true, true, 2>(p, c) : run_fwd<T, FMT, D, true, true, 1>(p, c);
  return two ? run_fwd<T, FMT, D, true, false, 2>(p, c) : run_fwd<T, FMT, D, true, false, 1>(p, c);
}

}  // namespace

uint64_t attn_paged_workspace(const AttnProblem& p) {
  // a call with part of the plan's sequences and tokens needs no more: its
  // units have at most as many rows
  const AttnGeom& g = p.geom;
  return ((fwd_counter_bytes(g) + 255u) & ~255ull) +
         2u * kFwdMaxCtas * static_cast<uint64_t>(fwd_part_floats(fwd_part_rows(g), p.dim)) * 4u;
}

std::string attn_forward_name(const AttnProblem& p) {
  const AttnGeom& g = p.geom;
  std::string s = std::string("attn_fwd_kernel<") + (p.dtype == GPO_BFLOAT16 ? "bf16" : "f16") +
                  ",D=" + std::to_string(p.dim) + (p.paged ? ",paged" : ",dense") +
                  ",tiles=" + std::to_string(fwd_tiles(g));
  if (p.paged && fwd_is_cut(g)) s += ",cut";
  if (!p.paged && attn_has_unseen(g)) s += ",unseen";
  return s + ">";
}

gpo_status launch_attn_forward(const AttnProblem& p, const LaunchCtx& c) {
  if (p.dtype == GPO_BFLOAT16)
    return p.dim == 128 ? run_fwd_form<__nv_bfloat16, 1, 128>(p, c)
                        : run_fwd_form<__nv_bfloat16, 1, 64>(p, c);
  return p.dim == 128 ? run_fwd_form<__half, 0, 128>(p, c) : run_fwd_form<__half, 0, 64>(p, c);
}

}  // namespace gpo
