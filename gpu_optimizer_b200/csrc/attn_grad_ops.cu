// Gradient of attention with a sliding window and sink tokens (sm_100a,
// tcgen05): dQ, dK, dV from dO, the inputs and the forward's O and
// log-sum-exp L.
//
//   P  = exp(scale Q K^T - L)        delta = sum_d dO * O
//   dV = P^T dO                      dS = P * (dO V^T - delta)
//   dQ = scale dS K                  dK = scale dS^T Q
// with dK and dV summed over the query heads of a kv head.
//
// Three kernels: the rows' statistics (memory bound), dK and dV by key tile
// and dQ by query tile.  The scores are computed in both of the latter (7
// products in place of 5), because each sum then has one owner and a fixed
// order: no atomics, equal inputs give equal bits, and no fp32 copy of dQ
// goes through memory.  P and dS are rounded to the inputs' type as MMA
// operands; every sum is fp32 in TMEM.
#include <algorithm>

#include "attn_ops.cuh"

namespace gpo {

constexpr int kGradStages = 2;
constexpr int kGradThreads = 384;  // 4 service warps, 2 x 4 elementwise warps
constexpr int kGradEwWarps = 8;

struct GradArgs {
  AttnGeom geom;
  // per packed row: -L in the log2 domain, and delta; 128 + 128 floats per
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
  int kv_tiles;    // key tiles of a head
  int sink_tiles;  // of them, tiles with a sink key
  int far_tiles;   // query tiles of a far piece (see kv_piece)
  int far_pieces;  // far pieces of a sink tile
  int items;
  unsigned int* err;
};

__device__ __forceinline__ float* grad_stats(const GradArgs& a, int b, int h, int tile) {
  return a.stats + ((static_cast<int64_t>(b) * a.geom.heads_kv + h) * a.geom.tiles + tile) * 256;
}

// ---------------------------------------------------------------- row stats
// One block per (query tile, kv head, batch); D / 8 lanes read a row of O
// and dO as 16-byte vectors.
template <typename T, int D>
__global__ void __launch_bounds__(256) attn_grad_stats_kernel(const GradArgs a) {
  const AttnGeom& g = a.geom;
  constexpr int LPR = D / 8, RPW = 32 / LPR;  // lanes per row, rows per warp
  const int tile = blockIdx.x % g.tiles, bh = blockIdx.x / g.tiles;
  const int h = bh % g.heads_kv, b = bh / g.heads_kv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* st = grad_stats(a, b, h, tile);
#pragma unroll 4
  for (int r0 = warp * 16; r0 < warp * 16 + 16; r0 += RPW) {
    const int r = r0 + lane / LPR;
    const int token = tile * g.tpt + r / g.g, head = h * g.g + r % g.g;
    const bool live = r < g.tpt * g.g && token < g.q_len;
    float s = 0.f;
    if (live) {
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
        const float l = a.lse[(static_cast<int64_t>(b) * g.q_len + token) *
                                  (static_cast<int64_t>(g.heads_kv) * g.g) + head];
        // a row that saw no key (L = -inf) has P = 0 everywhere, too
        nl = l == -INFINITY ? -INFINITY : -l * 1.4426950408889634f;
      }
      st[r] = nl;
      st[128 + r] = live ? s : 0.f;
    }
  }
}

// ------------------------------------------------------------- shared parts
struct GradShared {
  uint64_t own_full, own_empty;                            // the item's own two tiles
  uint64_t in_full[kGradStages], in_empty[kGradStages];    // ring of the other side
  uint64_t s_full[2], dp_full;
  uint64_t p_ready, ds_ready;
  uint64_t acc_full, acc_free;
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
};

__device__ __forceinline__ void grad_init(GradShared& sh) {
  mbar_init(smem_u32(&sh.own_full), 1);
  mbar_init(smem_u32(&sh.own_empty), 1);
  for (int s = 0; s < kGradStages; ++s) {
    mbar_init(smem_u32(&sh.in_full[s]), 1);
    mbar_init(smem_u32(&sh.in_empty[s]), 1);
  }
  mbar_init(smem_u32(&sh.s_full[0]), 1);
  mbar_init(smem_u32(&sh.s_full[1]), 1);
  mbar_init(smem_u32(&sh.dp_full), 1);
  mbar_init(smem_u32(&sh.p_ready), kGradEwWarps);
  mbar_init(smem_u32(&sh.ds_ready), kGradEwWarps);
  mbar_init(smem_u32(&sh.acc_full), 1);
  mbar_init(smem_u32(&sh.acc_free), kGradEwWarps);
  mbar_init(smem_u32(&sh.drain), 1);
  sh.abort = 0;
  fence_barrier_init();
}

struct GradRing {
  int slot = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void step() {
    if (++slot == kGradStages) {
      slot = 0;
      parity ^= 1u;
    }
  }
};

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
__device__ __forceinline__ void store_row(uint32_t taddr, T* dst, float f, bool live, bool zero) {
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
#pragma unroll
    for (int i = 0; i < 4; ++i)
      reinterpret_cast<uint4*>(dst + c * 32)[i] =
          make_uint4(pk[4 * i], pk[4 * i + 1], pk[4 * i + 2], pk[4 * i + 3]);
  }
}

// ------------------------------------------------------------------ dK, dV
// Key tile kt is seen by the query tiles [first, last].  For a tile with
// sink keys these are: the tiles of its window (the main piece), and all
// later ones, which see the sink keys alone; those are cut into far pieces
// of far_tiles query tiles, so that no CTA has a longer way than the others.
// The pieces' sums of the sink rows are joined by attn_grad_join_kernel.
struct KvPiece {
  int b, h, kt, piece;  // piece 0: main
  int first, n;         // query tiles
};

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

template <typename T, int FMT, int D>
__global__ void __launch_bounds__(kGradThreads, 1)
    attn_grad_kv_kernel(const __grid_constant__ CUtensorMap tma_q,
                        const __grid_constant__ CUtensorMap tma_do,
                        const __grid_constant__ CUtensorMap tma_k,
                        const __grid_constant__ CUtensorMap tma_v,
                        const __grid_constant__ GradArgs args) {
  constexpr uint32_t TILE = 128u * D * 2;        // bytes of a 128-row tile
  constexpr uint32_t STAGE = 2 * TILE + 1024u;   // Q, dO, statistics
  constexpr uint32_t IDESC_S = make_idesc(FMT, 128, 128, false, false);
  constexpr uint32_t IDESC_O = make_idesc(FMT, 128, D, false, true);
  constexpr uint32_t S_COL = 0, DP_COL = 128, DV_COL = 256, DK_COL = 256 + D;

  __shared__ GradShared sh;
  extern __shared__ uint8_t dyn_smem[];
  const uint32_t base = (smem_u32(dyn_smem) + 1023u) & ~1023u;
  const uint32_t k_smem = base, v_smem = base + TILE, ring = base + 2 * TILE;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const AttnGeom& g = args.geom;
  unsigned int* err = args.err;

  if (threadIdx.x == 0) {
    grad_init(sh);
    tma_prefetch_desc(&tma_q);
    tma_prefetch_desc(&tma_do);
    tma_prefetch_desc(&tma_k);
    tma_prefetch_desc(&tma_v);
  }
  // rows of a query tile that hold no query (128 is not a multiple of g):
  // no copy writes them, and 0 * (what was there) need not be 0
  {
    const int unused = 128 - g.tpt * g.g;
    const int vecs = unused * 8 * (D / 64);
    for (int i = threadIdx.x; i < kGradStages * 2 * vecs; i += kGradThreads) {
      const int s = i / (2 * vecs), m = i / vecs % 2, e = i % vecs;
      const int atom = e / (unused * 8), x = e % (unused * 8);
      asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                       ring + s * STAGE + m * TILE + atom * 128 * 128 +
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
  volatile int* abort_flag = &sh.abort;

  if (warp == 0 && lane == 0) {
    // -------------------------------------------------------- producer
    const uint32_t rows_bytes = static_cast<uint32_t>(g.tpt * g.g) * D * 2;
    bool ok = true;
    int issued = 0, own = 0;
    GradRing pos;
    for (int item = blockIdx.x; item < args.items && ok; item += gridDim.x) {
      const KvPiece p = kv_piece(args, item);
      if (p.n == 0) continue;
      ok = own == 0 || mbar_wait(smem_u32(&sh.own_empty), (own - 1) & 1u, abort_flag, err,
                                 kErrWaitProducer);
      if (!ok) break;
      mbar_arrive_expect_tx(smem_u32(&sh.own_full), 2 * TILE);
      for (int c = 0; c < D / 64; ++c) {
        tma_load_4d(k_smem + c * 128 * 128, &tma_k, smem_u32(&sh.own_full), c * 64, p.h,
                    p.kt * 128, p.b);
        tma_load_4d(v_smem + c * 128 * 128, &tma_v, smem_u32(&sh.own_full), c * 64, p.h,
                    p.kt * 128, p.b);
      }
      ++own;
      for (int j = 0; j < p.n; ++j) {
        if (!mbar_wait(smem_u32(&sh.in_empty[pos.slot]), pos.parity ^ 1u, abort_flag, err,
                       kErrWaitProducer)) {
          ok = false;
          break;
        }
        const uint32_t bar = smem_u32(&sh.in_full[pos.slot]);
        const uint32_t dst = ring + pos.slot * STAGE;
        const int tile = p.first + j;
        mbar_arrive_expect_tx(bar, 2 * rows_bytes + 1024u);
        for (int c = 0; c < D / 64; ++c) {
          tma_load_5d(dst + c * 128 * 128, &tma_q, bar, c * 64, 0, p.h, tile * g.tpt, p.b);
          tma_load_5d(dst + TILE + c * 128 * 128, &tma_do, bar, c * 64, 0, p.h, tile * g.tpt,
                      p.b);
        }
        bulk_load(dst + 2 * TILE, grad_stats(args, p.b, p.h, tile), 1024u, bar);
        ++issued;
        pos.step();
      }
    }
    if (!ok) {
      if (own > 0) mbar_wait_drain(smem_u32(&sh.own_full), (own - 1) & 1u, err);
      for (int j = max(0, issued - kGradStages); j < issued; ++j)
        mbar_wait_drain(smem_u32(&sh.in_full[j % kGradStages]), (j / kGradStages) & 1u, err);
    }
  } else if (warp == 1 && lane == 0) {
    // ------------------------------------------------------ MMA issuer
    // S(j+1) follows dV(j), which reads P(j) in the same columns, and
    // dP(j+1) follows dK(j) in the same way: MMAs run in issue order.
    auto wait = [&](const uint64_t* bar, uint32_t parity) {
      const uint32_t b = smem_u32(bar);
      return mbar_test_wait(b, parity) || mbar_wait(b, parity, abort_flag, err, kErrWaitMma);
    };
    const uint32_t k_lo = smem_desc_lo(k_smem, 16), v_lo = smem_desc_lo(v_smem, 16);
    bool ok = true;
    GradRing pos;
    uint32_t own = 0, cnt = 0;  // items, query tiles so far
    for (int item = blockIdx.x; item < args.items && ok; item += gridDim.x) {
      const KvPiece p = kv_piece(args, item);
      if (p.n == 0) continue;
      ok = wait(&sh.own_full, own & 1u) && wait(&sh.in_full[pos.slot], pos.parity);
      if (!ok) break;
      {
        const uint32_t q = ring + pos.slot * STAGE;
        mma_rows<D>(tmem + S_COL, k_lo, smem_desc_lo(q, 16), IDESC_S);
        mma_commit(smem_u32(&sh.s_full[0]));
        mma_rows<D>(tmem + DP_COL, v_lo, smem_desc_lo(q + TILE, 16), IDESC_S);
        mma_commit(smem_u32(&sh.dp_full));
      }
      // the previous item's sums have been read out of TMEM
      if (own > 0) ok = wait(&sh.acc_free, (own - 1) & 1u);
      for (int j = 0; j < p.n && ok; ++j, ++cnt) {
        const uint32_t q = ring + pos.slot * STAGE;
        GradRing nxt = pos;
        nxt.step();
        const uint32_t qn = ring + nxt.slot * STAGE;
        ok = wait(&sh.p_ready, cnt & 1u);
        if (!ok) break;
        tc_fence_after();
        mma_cols(tmem + DV_COL, tmem + S_COL, smem_desc_lo(q + TILE, 128 * 128), IDESC_O, j == 0);
        if (j + 1 < p.n) {
          ok = wait(&sh.in_full[nxt.slot], nxt.parity);
          if (!ok) break;
          mma_rows<D>(tmem + S_COL, k_lo, smem_desc_lo(qn, 16), IDESC_S);
          mma_commit(smem_u32(&sh.s_full[0]));
        }
        ok = wait(&sh.ds_ready, cnt & 1u);
        if (!ok) break;
        tc_fence_after();
        mma_cols(tmem + DK_COL, tmem + DP_COL, smem_desc_lo(q, 128 * 128), IDESC_O, j == 0);
        mma_commit(smem_u32(&sh.in_empty[pos.slot]));
        if (j + 1 < p.n) {
          mma_rows<D>(tmem + DP_COL, v_lo, smem_desc_lo(qn + TILE, 16), IDESC_S);
          mma_commit(smem_u32(&sh.dp_full));
        } else {
          mma_commit(smem_u32(&sh.acc_full));
          mma_commit(smem_u32(&sh.own_empty));
        }
        pos = nxt;
      }
      ++own;
    }
    if (!ok) {
      mma_commit(smem_u32(&sh.drain));
      mbar_wait_drain(smem_u32(&sh.drain), 0, err);
    }
  } else if (warp >= 4) {
    // ------------------------- elementwise: thread = key, 64 packed rows
    const int wg = (warp - 4) >> 2, q = warp & 3;
    const int row = q * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t s_t = tmem + lane_addr + S_COL + wg * 64;
    const uint32_t dp_t = tmem + lane_addr + DP_COL + wg * 64;
    const float2 scale2 = make_float2(args.scale_log2, args.scale_log2);
    const int off = g.kv_len - g.q_len;
    bool ok = true;
    GradRing pos;
    uint32_t own = 0, cnt = 0;
    auto wait = [&](const uint64_t* bar, uint32_t parity) {
      return __all_sync(0xffffffffu,
                        mbar_wait(smem_u32(bar), parity, abort_flag, err, kErrWaitSoftmax));
    };
    auto release = [&](uint64_t* bar) {
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(bar));
    };
    for (int item = blockIdx.x; item < args.items && ok; item += gridDim.x) {
      const KvPiece p = kv_piece(args, item);
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
        // statistics are written by the bulk copy that in_full counts
        ok = wait(&sh.in_full[pos.slot], pos.parity) && wait(&sh.s_full[0], cnt & 1u);
        if (!ok) break;
        tc_fence_after();
        const uint32_t st = ring + pos.slot * STAGE + 2 * TILE + wg * 256;
        float pr[64];
#pragma unroll
        for (int c = 0; c < 2; ++c)
          tmem_ld32(s_t + c * 32, *reinterpret_cast<uint32_t(*)[32]>(
                                      reinterpret_cast<uint32_t*>(pr) + c * 32));
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 64; i += 4) {
          float4 nl;
          asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(nl.x), "=f"(nl.y), "=f"(nl.z), "=f"(nl.w)
                       : "r"(st + i * 4));
          const float2 x = __ffma2_rn(make_float2(pr[i], pr[i + 1]), scale2,
                                      make_float2(nl.x, nl.y));
          const float2 y = __ffma2_rn(make_float2(pr[i + 2], pr[i + 3]), scale2,
                                      make_float2(nl.z, nl.w));
          pr[i] = ex2_approx(x.x);
          pr[i + 1] = ex2_approx(x.y);
          pr[i + 2] = ex2_approx(y.x);
          pr[i + 3] = ex2_approx(y.y);
        }
        if (masked) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint32_t see = bits_below(c_hi, c) & ~bits_below(c_lo, c);
#pragma unroll
            for (int i = 0; i < 32; ++i) pr[c * 32 + i] = (see & (1u << i)) ? pr[c * 32 + i] : 0.f;
          }
        }
        {
          uint32_t pk[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) pk[i] = pack2<FMT>(pr[2 * i], pr[2 * i + 1]);
          tmem_st32(s_t, pk);
        }
        release(&sh.p_ready);
        ok = wait(&sh.dp_full, cnt & 1u);
        if (!ok) break;
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
                         : "r"(st + 512 + (c * 32 + i) * 4));
            const float d[4] = {dl.x, dl.y, dl.z, dl.w};
            float ds[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const float pv = pr[c * 32 + i + u];
              ds[u] = pv * (__uint_as_float(dp[i + u]) - d[u]);
            }
            pk[c * 16 + i / 2] = pack2<FMT>(ds[0], ds[1]);
            pk[c * 16 + i / 2 + 1] = pack2<FMT>(ds[2], ds[3]);
          }
        }
        if (masked) {
          // 0 * (dP - delta) is not 0 when the masked dP is not finite
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const uint32_t see = (bits_below(c_hi, i / 16) & ~bits_below(c_lo, i / 16)) >>
                                 (2 * (i % 16));
            pk[i] &= ((see & 1u) ? 0x0000ffffu : 0u) | ((see & 2u) ? 0xffff0000u : 0u);
          }
        }
        tmem_st32(dp_t, pk);
        release(&sh.ds_ready);
        pos.step();
      }
      if (!ok) break;
      if (p.n > 0) {
        ok = wait(&sh.acc_full, own & 1u);
        if (!ok) break;
        tc_fence_after();
      }
      // warpgroup 0 writes dV, warpgroup 1 dK
      const uint32_t acc = tmem + lane_addr + (wg == 0 ? DV_COL : DK_COL);
      const float f = wg == 0 ? 1.f : args.scale;
      const bool sink = key < g.sinks;
      T* dst = wg == 0 ? static_cast<T*>(args.dv) + p.b * args.dv_batch + key * args.dv_token +
                             p.h * args.dv_head
                       : static_cast<T*>(args.dk) + p.b * args.dk_batch + key * args.dk_token +
                             p.h * args.dk_head;
      if (k0 < g.sinks) {
        float* part = sink ? kv_partial<D>(args, p.b, p.h, key, p.piece) + wg * D : nullptr;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t r[32];
          tmem_ld32(acc + c * 32, r);
          tmem_wait_ld();
          if (sink && key < g.kv_len) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<float4*>(part + c * 32 + i) =
                  p.n == 0 ? make_float4(0.f, 0.f, 0.f, 0.f)
                           : make_float4(__uint_as_float(r[i]) * f, __uint_as_float(r[i + 1]) * f,
                                         __uint_as_float(r[i + 2]) * f,
                                         __uint_as_float(r[i + 3]) * f);
          }
        }
      }
      if (p.piece == 0)
        store_row<T, FMT, D>(acc, dst, f, key < g.kv_len && !sink, p.n == 0);
      if (p.n > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.acc_free));
        ++own;
      }
    }
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

// ---------------------------------------------------------------------- dQ
template <typename T, int FMT, int D>
__global__ void __launch_bounds__(kGradThreads, 1)
    attn_grad_q_kernel(const __grid_constant__ CUtensorMap tma_q,
                       const __grid_constant__ CUtensorMap tma_do,
                       const __grid_constant__ CUtensorMap tma_k,
                       const __grid_constant__ CUtensorMap tma_v,
                       const __grid_constant__ GradArgs args) {
  constexpr uint32_t TILE = 128u * D * 2;
  constexpr uint32_t STAGE = 2 * TILE;  // K, V
  constexpr uint32_t IDESC_S = make_idesc(FMT, 128, 128, false, false);
  constexpr uint32_t IDESC_O = make_idesc(FMT, 128, D, false, true);
  // two S buffers (dS overlays S), dP, dQ
  constexpr uint32_t S_COL = 0, DP_COL = 256, DQ_COL = 384;

  __shared__ GradShared sh;
  extern __shared__ uint8_t dyn_smem[];
  const uint32_t base = (smem_u32(dyn_smem) + 1023u) & ~1023u;
  const uint32_t q_smem = base, do_smem = base + TILE, ring = base + 2 * TILE;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const AttnGeom& g = args.geom;
  unsigned int* err = args.err;
  const AttnSeq seq{g.q_len, g.kv_len, 0, g.kv_len - g.q_len};

  if (threadIdx.x == 0) {
    grad_init(sh);
    tma_prefetch_desc(&tma_q);
    tma_prefetch_desc(&tma_do);
    tma_prefetch_desc(&tma_k);
    tma_prefetch_desc(&tma_v);
  }
  if (warp == 2) {
    tmem_alloc(smem_u32(&sh.tmem_base), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem_base;
  volatile int* abort_flag = &sh.abort;

  struct Item {
    int b, h, t0, t1, tile;
    AttnBlocks blk;
  };
  auto item_of = [&](int item) {
    Item it;
    it.h = item % g.heads_kv;
    const int r = item / g.heads_kv;
    it.b = r % g.batch;
    it.tile = g.tiles - 1 - r / g.batch;  // the longest rows first
    it.t0 = it.tile * g.tpt;
    it.t1 = min(it.t0 + g.tpt, g.q_len);
    it.blk = attn_blocks(g, seq, it.t0, it.t1);
    return it;
  };
  const int items = g.tiles * g.batch * g.heads_kv;

  if (warp == 0 && lane == 0) {
    const uint32_t rows_bytes = static_cast<uint32_t>(g.tpt * g.g) * D * 2;
    bool ok = true;
    int issued = 0, own = 0;
    GradRing pos;
    for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
      const Item it = item_of(item);
      if (it.blk.n == 0) continue;
      ok = own == 0 || mbar_wait(smem_u32(&sh.own_empty), (own - 1) & 1u, abort_flag, err,
                                 kErrWaitProducer);
      if (!ok) break;
      mbar_arrive_expect_tx(smem_u32(&sh.own_full), 2 * rows_bytes);
      for (int c = 0; c < D / 64; ++c) {
        tma_load_5d(q_smem + c * 128 * 128, &tma_q, smem_u32(&sh.own_full), c * 64, 0, it.h,
                    it.t0, it.b);
        tma_load_5d(do_smem + c * 128 * 128, &tma_do, smem_u32(&sh.own_full), c * 64, 0, it.h,
                    it.t0, it.b);
      }
      ++own;
      for (int j = 0; j < it.blk.n; ++j) {
        if (!mbar_wait(smem_u32(&sh.in_empty[pos.slot]), pos.parity ^ 1u, abort_flag, err,
                       kErrWaitProducer)) {
          ok = false;
          break;
        }
        const uint32_t bar = smem_u32(&sh.in_full[pos.slot]);
        const uint32_t dst = ring + pos.slot * STAGE;
        mbar_arrive_expect_tx(bar, STAGE);
        for (int c = 0; c < D / 64; ++c) {
          tma_load_4d(dst + c * 128 * 128, &tma_k, bar, c * 64, it.h, it.blk.at(j) * 128, it.b);
          tma_load_4d(dst + TILE + c * 128 * 128, &tma_v, bar, c * 64, it.h, it.blk.at(j) * 128,
                      it.b);
        }
        ++issued;
        pos.step();
      }
    }
    if (!ok) {
      if (own > 0) mbar_wait_drain(smem_u32(&sh.own_full), (own - 1) & 1u, err);
      for (int j = max(0, issued - kGradStages); j < issued; ++j)
        mbar_wait_drain(smem_u32(&sh.in_full[j % kGradStages]), (j / kGradStages) & 1u, err);
    }
  } else if (warp == 1 && lane == 0) {
    // S(j+1) goes to the other buffer before dS(j) is waited for; dP(j+1)
    // then has its columns back (they are read by the time dS(j) is ready)
    // and comes before dQ(j), so that the elementwise warps wait least.
    auto wait = [&](const uint64_t* bar, uint32_t parity) {
      const uint32_t b = smem_u32(bar);
      return mbar_test_wait(b, parity) || mbar_wait(b, parity, abort_flag, err, kErrWaitMma);
    };
    const uint32_t q_lo = smem_desc_lo(q_smem, 16), do_lo = smem_desc_lo(do_smem, 16);
    bool ok = true;
    GradRing pos;
    uint32_t own = 0, cnt = 0;
    for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
      const Item it = item_of(item);
      const int n = it.blk.n;
      if (n == 0) continue;
      ok = wait(&sh.own_full, own & 1u) && wait(&sh.in_full[pos.slot], pos.parity);
      if (!ok) break;
      {
        const uint32_t k = ring + pos.slot * STAGE;
        mma_rows<D>(tmem + S_COL + (cnt & 1u) * 128, q_lo, smem_desc_lo(k, 16), IDESC_S);
        mma_commit(smem_u32(&sh.s_full[cnt & 1u]));
        mma_rows<D>(tmem + DP_COL, do_lo, smem_desc_lo(k + TILE, 16), IDESC_S);
        mma_commit(smem_u32(&sh.dp_full));
      }
      if (own > 0) ok = wait(&sh.acc_free, (own - 1) & 1u);
      for (int j = 0; j < n && ok; ++j, ++cnt) {
        const uint32_t k = ring + pos.slot * STAGE;
        GradRing nxt = pos;
        nxt.step();
        const uint32_t kn = ring + nxt.slot * STAGE;
        if (j + 1 < n) {
          ok = wait(&sh.in_full[nxt.slot], nxt.parity);
          if (!ok) break;
          mma_rows<D>(tmem + S_COL + ((cnt + 1) & 1u) * 128, q_lo, smem_desc_lo(kn, 16), IDESC_S);
          mma_commit(smem_u32(&sh.s_full[(cnt + 1) & 1u]));
        }
        ok = wait(&sh.ds_ready, cnt & 1u);
        if (!ok) break;
        tc_fence_after();
        if (j + 1 < n) {
          mma_rows<D>(tmem + DP_COL, do_lo, smem_desc_lo(kn + TILE, 16), IDESC_S);
          mma_commit(smem_u32(&sh.dp_full));
        } else {
          mma_commit(smem_u32(&sh.own_empty));
        }
        mma_cols(tmem + DQ_COL, tmem + S_COL + (cnt & 1u) * 128, smem_desc_lo(k, 128 * 128),
                 IDESC_O, j == 0);
        mma_commit(smem_u32(&sh.in_empty[pos.slot]));
        if (j + 1 == n) mma_commit(smem_u32(&sh.acc_full));
        pos = nxt;
      }
      ++own;
    }
    if (!ok) {
      mma_commit(smem_u32(&sh.drain));
      mbar_wait_drain(smem_u32(&sh.drain), 0, err);
    }
  } else if (warp >= 4) {
    // --------------------- elementwise: thread = packed row, 64 keys
    const int wg = (warp - 4) >> 2, q = warp & 3;
    const int row = q * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t dp_t = tmem + lane_addr + DP_COL + wg * 64;
    const float2 scale2 = make_float2(args.scale_log2, args.scale_log2);
    const int row_token = row / g.g, row_head = row % g.g;
    bool ok = true;
    uint32_t own = 0, cnt = 0;
    auto wait = [&](const uint64_t* bar, uint32_t parity) {
      return __all_sync(0xffffffffu,
                        mbar_wait(smem_u32(bar), parity, abort_flag, err, kErrWaitSoftmax));
    };
    for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
      const Item it = item_of(item);
      const int token = it.t0 + row_token;
      const bool live = row_token < g.tpt && token < it.t1;
      const float* st = grad_stats(args, it.b, it.h, it.tile);
      const float nl = st[row], delta = st[128 + row];
      const float2 shift2 = make_float2(nl, nl);
      for (int j = 0; j < it.blk.n; ++j, ++cnt) {
        const int key0 = it.blk.at(j) * 128;
        const bool masked = block_is_masked(g, seq, it.t0, it.t1, key0);
        const RowMask rm = row_mask(g, token + seq.off, key0 + wg * 64);
        const uint32_t s_t = tmem + lane_addr + S_COL + (cnt & 1u) * 128 + wg * 64;
        ok = wait(&sh.s_full[cnt & 1u], (cnt >> 1) & 1u);
        if (!ok) break;
        tc_fence_after();
        float pr[64];
#pragma unroll
        for (int c = 0; c < 2; ++c)
          tmem_ld32(s_t + c * 32, *reinterpret_cast<uint32_t(*)[32]>(
                                      reinterpret_cast<uint32_t*>(pr) + c * 32));
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 64; i += 2) {
          const float2 x = __ffma2_rn(make_float2(pr[i], pr[i + 1]), scale2, shift2);
          pr[i] = ex2_approx(x.x);
          pr[i + 1] = ex2_approx(x.y);
        }
        ok = wait(&sh.dp_full, cnt & 1u);
        if (!ok) break;
        tc_fence_after();
        uint32_t pk[32];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t dp[32];
          tmem_ld32(dp_t + c * 32, dp);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; i += 2)
            pk[c * 16 + i / 2] =
                pack2<FMT>(pr[c * 32 + i] * (__uint_as_float(dp[i]) - delta),
                           pr[c * 32 + i + 1] * (__uint_as_float(dp[i + 1]) - delta));
          if (masked) {
            const uint32_t see = rm.word(c);
#pragma unroll
            for (int i = 0; i < 16; ++i)
              pk[c * 16 + i] &= ((see & (1u << (2 * i))) ? 0x0000ffffu : 0u) |
                                ((see & (2u << (2 * i))) ? 0xffff0000u : 0u);
          }
        }
        tmem_st32(s_t, pk);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.ds_ready));
      }
      if (!ok) break;
      if (it.blk.n > 0) {
        ok = wait(&sh.acc_full, own & 1u);
        if (!ok) break;
        tc_fence_after();
      }
      // each warpgroup writes half of the dims
      T* dst = static_cast<T*>(args.dq) + it.b * args.dq_batch + token * args.dq_token +
               (it.h * g.g + row_head) * args.dq_head + wg * (D / 2);
      store_row<T, FMT, D / 2>(tmem + lane_addr + DQ_COL + wg * (D / 2), dst, args.scale, live,
                               it.blk.n == 0);
      if (it.blk.n > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.acc_free));
        ++own;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2) tmem_dealloc(tmem, 512);
}

// ------------------------------------------------------------------- host
namespace {

struct GradPlan {
  int kv_tiles, sink_tiles, far_tiles, far_pieces;
  uint64_t stats_bytes, partial_bytes;
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
    p.far_pieces = next >= g.tiles ? 0 : static_cast<int>(cdiv(g.tiles - next, p.far_tiles));
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
  if (!encode_rows_map(&mq, p.dtype, p.q, D, g.g, g.tpt) ||
      !encode_rows_map(&mdo, p.dtype, gp.dout, D, g.g, g.tpt) ||
      !encode_keys_map(&mk, p.dtype, p.k, D, 128) || !encode_keys_map(&mv, p.dtype, p.v, D, 128))
    return GPO_BAD_ARGS;
  const GradPlan pl = grad_plan(g, D);
  GradArgs a{};
  a.geom = g;
  a.stats = static_cast<float*>(gp.workspace);
  a.partial = reinterpret_cast<float*>(static_cast<char*>(gp.workspace) + pl.stats_bytes);
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
  a.scale = p.scale;
  a.scale_log2 = p.scale * 1.4426950408889634f;
  a.kv_tiles = pl.kv_tiles;
  a.sink_tiles = pl.sink_tiles;
  a.far_tiles = pl.far_tiles;
  a.far_pieces = pl.far_pieces;
  a.err = c.err;
  const int64_t heads = static_cast<int64_t>(g.batch) * g.heads_kv;
  const int64_t q_items = heads * g.tiles;
  const int64_t kv_items = heads * (pl.kv_tiles + static_cast<int64_t>(pl.sink_tiles) * pl.far_pieces);
  const int64_t most = (1ll << 31) - 1024;
  if (q_items > most || kv_items > most || heads * g.sinks > most) return GPO_BAD_ARGS;
  a.items = static_cast<int>(kv_items);
  const int sms = c.sm_count > 0 ? c.sm_count : 148;
  if (q_items > 0) {
    attn_grad_stats_kernel<T, D><<<static_cast<unsigned>(q_items), 256, 0, c.stream>>>(a);
    if (launch_status() != GPO_OK) return GPO_LAUNCH_ERROR;
  }
  constexpr uint32_t tile = 128u * D * 2u;
  if (kv_items > 0) {
    constexpr uint32_t dyn = 2 * tile + kGradStages * (2 * tile + 1024u) + 1024u;
    auto kern = attn_grad_kv_kernel<T, FMT, D>;
    const gpo_status s = ensure_smem_attr(reinterpret_cast<const void*>(kern), dyn);
    if (s != GPO_OK) return s;
    kern<<<static_cast<unsigned>(std::min<int64_t>(kv_items, sms)), kGradThreads, dyn,
           c.stream>>>(mq, mdo, mk, mv, a);
    if (launch_status() != GPO_OK) return GPO_LAUNCH_ERROR;
    if (pl.sink_tiles > 0) {
      attn_grad_join_kernel<T, D>
          <<<static_cast<unsigned>(heads * g.sinks), 2 * D, 0, c.stream>>>(a);
      if (launch_status() != GPO_OK) return GPO_LAUNCH_ERROR;
    }
  }
  if (q_items > 0) {
    constexpr uint32_t dyn = 2 * tile + kGradStages * 2 * tile + 1024u;
    auto kern = attn_grad_q_kernel<T, FMT, D>;
    const gpo_status s = ensure_smem_attr(reinterpret_cast<const void*>(kern), dyn);
    if (s != GPO_OK) return s;
    kern<<<static_cast<unsigned>(std::min<int64_t>(q_items, sms)), kGradThreads, dyn,
           c.stream>>>(mq, mdo, mk, mv, a);
  }
  return launch_status();
}

}  // namespace

uint64_t attn_grad_workspace(const AttnProblem& p) {
  const GradPlan pl = grad_plan(p.geom, p.dim);
  return pl.stats_bytes + pl.partial_bytes;
}

gpo_status launch_attn_grad(const AttnProblem& p, const AttnGradProblem& gp, const LaunchCtx& c) {
  if (p.dtype == GPO_BFLOAT16)
    return p.dim == 128 ? run_grad<__nv_bfloat16, 1, 128>(p, gp, c)
                        : run_grad<__nv_bfloat16, 1, 64>(p, gp, c);
  return p.dim == 128 ? run_grad<__half, 0, 128>(p, gp, c) : run_grad<__half, 0, 64>(p, gp, c);
}

}  // namespace gpo
