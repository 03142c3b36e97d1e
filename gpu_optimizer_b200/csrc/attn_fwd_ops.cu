// Attention with a sliding window and sink tokens over grouped heads, from
// strided dense K/V or from a paged cache (sm_100a, tcgen05).
//
// O = softmax(scale * Q K^T over the visible keys) V and, per row, the
// log-sum-exp of its scaled scores.  One pass over the visible K/V blocks
// with the running maximum and sum of each row in registers.
//
// One CTA per SM works through tiles of 128 query rows (attn_ops.cuh: a
// tile packs all query heads of a kv head, so K/V is read once per kv head):
//   warp 0  TMA of Q and of the K ring
//   warp 3  TMA of the V ring; clears V rows behind a sequence's last key
//   warp 1  MMA issuer: S_j = Q K_j^T into TMEM buffer j % 3, two blocks
//           ahead of O += P_j V_j (P overlays S as 16-bit pairs)
//   warp 2  TMEM owner
//   warps 4-7  softmax: thread = query row = TMEM lane
// Only blocks with a visible key are loaded.  A page that ends inside a
// block is loaded as boxes of its own rows; boxes without a key are asked
// for outside the tensor, which TMA fills with zeros.
#include <algorithm>

#include "attn_ops.cuh"

namespace gpo {

constexpr int kFwdStages = 3;   // K slots and V slots
constexpr int kFwdSBufs = 3;    // S/P buffers in TMEM
constexpr int kFwdThreads = 256;
constexpr float kFwdRescale = 8.0f;  // see the softmax

struct FwdShared {
  uint64_t q_full, q_empty;
  uint64_t k_full[kFwdStages], k_empty[kFwdStages];
  uint64_t v_full[kFwdStages], v_empty[kFwdStages];
  uint64_t v_clean[kFwdStages];  // the slot's block has been cleared behind the last key
  uint64_t s_full[kFwdSBufs], p_full[kFwdSBufs], pv_done[kFwdSBufs];
  uint64_t o_full, o_free;
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
};

struct FwdArgs {
  AttnGeom geom;
  void* out;
  float* lse;  // (batch, q_len, heads) or (tokens, heads); may be null
  int64_t o_batch, o_token, o_head;
  float scale_log2;
  int items;
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

// One work item: a tile of query rows of one sequence and kv head.
struct FwdItem {
  int b, h, t0, t1;
  AttnSeq seq;
  AttnBlocks blk;
};

template <bool PAGED>
__device__ __forceinline__ FwdItem fwd_item(const FwdArgs& a, int item) {
  const AttnGeom& g = a.geom;
  FwdItem it;
  it.h = item % g.heads_kv;
  const int r = item / g.heads_kv;
  it.b = r % g.batch;
  const int tile = g.tiles - 1 - r / g.batch;  // the longest rows first
  it.seq = attn_seq<PAGED>(g, it.b, a.err);
  it.t0 = tile * g.tpt;
  it.t1 = min(it.t0 + g.tpt, it.seq.q_len);
  it.blk = attn_blocks(g, it.seq, it.t0, it.t1);
  return it;
}

template <typename T, int FMT, int D, bool PAGED>
__global__ void __launch_bounds__(kFwdThreads, 1)
    attn_fwd_kernel(const __grid_constant__ CUtensorMap tma_q,
                    const __grid_constant__ CUtensorMap tma_k,
                    const __grid_constant__ CUtensorMap tma_v,
                    const __grid_constant__ FwdArgs args) {
  constexpr int BN = kOpsBN;
  constexpr int SW = 128;               // swizzle atom: 64 dims of a row
  constexpr int ATOMS = D / 64;
  constexpr uint32_t Q_BYTES = 128u * D * 2;
  constexpr uint32_t KV_BYTES = static_cast<uint32_t>(BN) * D * 2;
  constexpr int NB = kFwdSBufs, LAG = NB - 1;
  constexpr uint32_t IDESC_S = make_idesc(FMT, 128, BN, false, false);
  constexpr uint32_t IDESC_O = make_idesc(FMT, 128, D, false, true);
  static_assert(D + NB * BN <= 512, "TMEM holds 512 columns");

  __shared__ FwdShared sh;
  extern __shared__ uint8_t dyn_smem[];
  const uint32_t base = (smem_u32(dyn_smem) + 1023u) & ~1023u;
  const uint32_t q_smem = base;
  const uint32_t k_smem = q_smem + Q_BYTES;
  const uint32_t v_smem = k_smem + kFwdStages * KV_BYTES;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const AttnGeom& g = args.geom;
  unsigned int* err = args.err;

  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&sh.q_full), 1);
    mbar_init(smem_u32(&sh.q_empty), 1);
    for (int s = 0; s < kFwdStages; ++s) {
      mbar_init(smem_u32(&sh.k_full[s]), 1);
      mbar_init(smem_u32(&sh.k_empty[s]), 1);
      mbar_init(smem_u32(&sh.v_full[s]), 1);
      mbar_init(smem_u32(&sh.v_empty[s]), 1);
      mbar_init(smem_u32(&sh.v_clean[s]), 1);
    }
    for (int b = 0; b < NB; ++b) {
      mbar_init(smem_u32(&sh.s_full[b]), 1);
      mbar_init(smem_u32(&sh.p_full[b]), 4);
      mbar_init(smem_u32(&sh.pv_done[b]), 1);
    }
    mbar_init(smem_u32(&sh.o_full), 1);
    mbar_init(smem_u32(&sh.o_free), 4);
    mbar_init(smem_u32(&sh.drain), 1);
    sh.abort = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tma_q);
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

  if (warp == 0 || warp == 3) {
    // ------------------------------------------- producers (K: 0, V: 3)
    // The whole warp runs the loop: each lane loads one box of a block.
    const bool is_k = warp == 0;
    const CUtensorMap* map = is_k ? &tma_k : &tma_v;
    const uint32_t ring = is_k ? k_smem : v_smem;
    uint64_t* full = is_k ? sh.k_full : sh.v_full;
    uint64_t* empty = is_k ? sh.k_empty : sh.v_empty;
    const int boxes = PAGED ? BN / g.box_rows : 1;
    bool ok = true;
    int issued = 0, q_loads = 0;
    RingPos2 pos;
    for (int item = blockIdx.x; item < args.items && ok; item += gridDim.x) {
      const FwdItem it = fwd_item<PAGED>(args, item);
      if (it.blk.n == 0) continue;
      if (is_k) {
        // Q of the previous item is free once its last S MMA is done
        ok = q_loads == 0 || mbar_wait(smem_u32(&sh.q_empty), (q_loads - 1) & 1u, abort_flag,
                                       err, kErrWaitProducer);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(smem_u32(&sh.q_full),
                                static_cast<uint32_t>(g.tpt * g.g) * D * 2);
#pragma unroll
          for (int c = 0; c < ATOMS; ++c)
            tma_load_5d(q_smem + c * 128 * SW, &tma_q, smem_u32(&sh.q_full), c * 64, 0, it.h,
                        it.seq.row0 + it.t0, PAGED ? 0 : it.b);
        }
        ++q_loads;
      }
      for (int i = 0; i < it.blk.n; ++i) {
        const int key0 = it.blk.at(i) * BN;
        int page = it.b, row = key0;
        if constexpr (PAGED) {
          const int key = key0 + lane * g.box_rows;
          page = g.num_pages;  // outside the tensor: zeros
          if (lane < boxes && key < it.seq.kv_len)
            page = __ldg(g.table + it.b * g.table_stride + key / g.page_size);
          row = key % g.page_size;
        }
        ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&empty[pos.slot]), pos.parity ^ 1u,
                                               abort_flag, err, kErrWaitProducer));
        if (!ok) break;
        const uint32_t bar = smem_u32(&full[pos.slot]);
        if (lane == 0) mbar_arrive_expect_tx(bar, KV_BYTES);
        __syncwarp();
        if (lane < boxes) {
          const uint32_t dst = ring + pos.slot * KV_BYTES +
                               static_cast<uint32_t>(PAGED ? lane * g.box_rows : 0) * SW;
#pragma unroll
          for (int c = 0; c < ATOMS; ++c)
            tma_load_4d(dst + c * BN * SW, map, bar, c * 64, it.h, row, page);
        }
        ++issued;
        if (PAGED && !is_k && key0 + BN > it.seq.kv_len) {
          // Slots behind a sequence's last key hold anything; P is 0 there,
          // but 0 * NaN is not: their V rows are cleared in shared memory
          // before the MMA reads the block (always an item's last one).
          ok = __all_sync(0xffffffffu,
                          mbar_wait(bar, pos.parity, abort_flag, err, kErrWaitProducer));
          if (!ok) break;
          for (int r = it.seq.kv_len - key0; r < BN; ++r)
            if (lane < ATOMS * 8)
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                               v_smem + pos.slot * KV_BYTES + (lane / 8) * BN * SW + r * SW +
                               (lane % 8) * 16),
                           "r"(0)
                           : "memory");
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sh.v_clean[pos.slot]));
        }
        pos.step(kFwdStages);
      }
    }
    if (!ok && lane == 0) {
      // let the copies in flight land before the CTA can exit
      if (q_loads > 0) mbar_wait_drain(smem_u32(&sh.q_full), (q_loads - 1) & 1u, err);
      for (int j = max(0, issued - kFwdStages); j < issued; ++j)
        mbar_wait_drain(smem_u32(&full[j % kFwdStages]), (j / kFwdStages) & 1u, err);
    }
  } else if (warp == 1 && lane == 0) {
    // ------------------------------------------------------- MMA issuer
    constexpr uint64_t HI = smem_desc_hi(8 * SW, SW);
    const uint32_t q_lo = smem_desc_lo(q_smem, 16);
    const uint32_t k_lo = smem_desc_lo(k_smem, 16);
    const uint32_t v_lo = smem_desc_lo(v_smem, BN * SW);
    bool ok = true;
    RingPos2 kpos, vpos, spos, ppos;
    uint32_t items_done = 0;
    uint32_t cleaned = 0;  // bit s: parity of slot s's next v_clean phase
    auto wait = [&](const uint64_t* bar, uint32_t parity) {
      return mbar_wait(smem_u32(bar), parity, abort_flag, err, kErrWaitMma);
    };
    for (int item = blockIdx.x; item < args.items && ok; item += gridDim.x) {
      const FwdItem it = fwd_item<PAGED>(args, item);
      const int n = it.blk.n;
      if (n == 0) continue;
      ok = wait(&sh.q_full, items_done & 1u);
      for (int i = 0; i < n + LAG && ok; ++i) {
        if (i < n) {
          // S buffer i % NB last held P of block i - NB, whose PV MMA was
          // issued before; MMAs of one thread execute in issue order
          ok = wait(&sh.k_full[kpos.slot], kpos.parity);
          if (!ok) break;
          tc_fence_after();
          const uint32_t s_tmem = tmem + D + spos.slot * BN;
          const uint32_t kd = k_lo + kpos.slot * (KV_BYTES >> 4);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = ((kk / 4) * 128 * SW + (kk % 4) * 32) >> 4;
            mma_f16_ss(s_tmem, HI | (q_lo + off), HI | (kd + off), IDESC_S, kk > 0 ? 1u : 0u);
          }
          mma_commit(smem_u32(&sh.s_full[spos.slot]));
          mma_commit(smem_u32(&sh.k_empty[kpos.slot]));
          if (i == n - 1) mma_commit(smem_u32(&sh.q_empty));
          kpos.step(kFwdStages);
          spos.step(NB);
        }
        const int j = i - LAG;
        if (j >= 0 && j < n) {
          ok = wait(&sh.v_full[vpos.slot], vpos.parity) &&
               wait(&sh.p_full[ppos.slot], ppos.parity);
          // the first PV overwrites O: the last item's epilogue has read it
          if (ok && j == 0 && items_done > 0) ok = wait(&sh.o_free, (items_done - 1) & 1u);
          if (PAGED && ok && (it.blk.at(j) + 1) * BN > it.seq.kv_len) {
            ok = wait(&sh.v_clean[vpos.slot], (cleaned >> vpos.slot) & 1u);
            cleaned ^= 1u << vpos.slot;
          }
          if (!ok) break;
          tc_fence_after();
          const uint32_t p_tmem = tmem + D + ppos.slot * BN;
          const uint32_t vd = v_lo + vpos.slot * (KV_BYTES >> 4);
#pragma unroll
          for (int kk = 0; kk < BN / 16; ++kk)
            mma_f16_ts(tmem, p_tmem + kk * 8, HI | (vd + ((kk * 16 * SW) >> 4)), IDESC_O,
                       (j > 0 || kk > 0) ? 1u : 0u);
          mma_commit(smem_u32(&sh.pv_done[ppos.slot]));
          mma_commit(smem_u32(&sh.v_empty[vpos.slot]));
          if (j == n - 1) mma_commit(smem_u32(&sh.o_full));
          vpos.step(kFwdStages);
          ppos.step(NB);
        }
      }
      ++items_done;
    }
    if (!ok) {
      mma_commit(smem_u32(&sh.drain));
      mbar_wait_drain(smem_u32(&sh.drain), 0, err);
    }
  } else if (warp >= 4) {
    // ------------------------------------------------ softmax, epilogue
    const int q = warp & 3;
    const int row = q * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t o_tmem = tmem + lane_addr;
    const float2 scale2 = make_float2(args.scale_log2, args.scale_log2);
    const int row_token = row / g.g, row_head = row % g.g;
    bool ok = true;
    RingPos2 spos, last_pv;
    uint32_t items_done = 0;
    for (int item = blockIdx.x; item < args.items && ok; item += gridDim.x) {
      const FwdItem it = fwd_item<PAGED>(args, item);
      if (it.t0 >= it.t1) continue;
      const int token = it.t0 + row_token;
      const bool live = row_token < g.tpt && token < it.t1;
      const int p = token + it.seq.off;
      float m_used = -INFINITY, l = 0.f;
      for (int j = 0; j < it.blk.n; ++j) {
        ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&sh.s_full[spos.slot]), spos.parity,
                                               abort_flag, err, kErrWaitSoftmax));
        if (!ok) break;
        if (q * 32 >= (it.t1 - it.t0) * g.g) {
          // no row of this warp holds a query (short chunks, single
          // tokens): whatever its P rows hold reaches only its own O rows
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sh.p_full[spos.slot]));
          spos.step(NB);
          continue;
        }
        tc_fence_after();
        const uint32_t sp = tmem + lane_addr + D + spos.slot * BN;
        uint32_t sv[BN];
#pragma unroll
        for (int c = 0; c < BN / 32; ++c)
          tmem_ld32(sp + c * 32, *reinterpret_cast<uint32_t(*)[32]>(sv + c * 32));
        tmem_wait_ld();
        auto f = [&](int i) { return __uint_as_float(sv[i]); };
        const int key0 = it.blk.at(j) * BN;
        if (block_is_masked(g, it.seq, it.t0, it.t1, key0)) {
          const RowMask rm = row_mask(g, p, key0);
#pragma unroll
          for (int i = 0; i < BN; ++i)
            if (!rm.sees(i)) sv[i] = __float_as_uint(-INFINITY);
        }
        float mx[4] = {f(0), f(1), f(2), f(3)};
#pragma unroll
        for (int i = 4; i + 1 < BN; i += 2)
          mx[(i >> 1) & 3] = fmax3(mx[(i >> 1) & 3], f(i), f(i + 1));
        const float mb = fmaxf(fmax3(mx[0], mx[1], mx[2]), mx[3]) * args.scale_log2;
        // The maximum that P is taken against moves only when a block's
        // exceeds it by 2^8 (or there is none yet): P <= 256 is as exact in
        // 16 bits as P <= 1, and O is rescaled in TMEM that rarely.
        if (j == 0) {
          m_used = mb;
        } else {
          const bool need = mb > m_used + kFwdRescale;
          if (__any_sync(0xffffffffu, need)) {
            // O holds the PV of every earlier block once the last is done
            ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&sh.pv_done[last_pv.slot]),
                                                   last_pv.parity, abort_flag, err,
                                                   kErrWaitSoftmax));
            if (!ok) break;
            tc_fence_after();
            const float m_new = need ? mb : m_used;
            const float alpha = need ? ex2_approx(m_used - m_new) : 1.f;
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t r[16];
              tmem_ld16(o_tmem + c * 16, r);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
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
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.p_full[spos.slot]));
        const float2 rsum = __fadd2_rn(__fadd2_rn(rs[0], rs[1]), __fadd2_rn(rs[2], rs[3]));
        l += rsum.x + rsum.y;
        last_pv = spos;
        spos.step(NB);
      }
      if (!ok) break;
      uint32_t ov[D];
      if (it.blk.n > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&sh.o_full), items_done & 1u, abort_flag,
                                               err, kErrWaitSoftmax));
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
          tmem_ld32(o_tmem + c * 32, *reinterpret_cast<uint32_t(*)[32]>(ov + c * 32));
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.o_free));
        ++items_done;
      } else {
#pragma unroll
        for (int i = 0; i < D; ++i) ov[i] = 0u;
      }
      if (live) {
        const int64_t r = it.seq.row0 + token;
        const int head = it.h * g.g + row_head;
        if (args.lse) {
          const int64_t at = (PAGED ? r : static_cast<int64_t>(it.b) * g.q_len + token) *
                                 (static_cast<int64_t>(g.heads_kv) * g.g) + head;
          args.lse[at] = l == 0.f ? -INFINITY : (m_used + log2f(l)) * 0.6931471805599453f;
        }
        const float inv_l = l == 0.f ? 0.f : 1.0f / l;
        T* orow = static_cast<T*>(args.out) + (PAGED ? 0 : it.b * args.o_batch) +
                  r * args.o_token + head * args.o_head;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          uint32_t pk[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float lo = __uint_as_float(ov[c * 8 + 2 * i]) * inv_l;
            const float hi = __uint_as_float(ov[c * 8 + 2 * i + 1]) * inv_l;
            pk[i] = FMT == 1 ? pack_bf16(lo, hi) : pack_f16(lo, hi);
          }
          reinterpret_cast<uint4*>(orow)[c] = make_uint4(pk[0], pk[1], pk[2], pk[3]);
        }
      }
    }
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

template <typename T, int FMT, int D, bool PAGED>
static gpo_status run_fwd(const AttnProblem& p, const LaunchCtx& c) {
  CUtensorMap mq, mk, mv;
  if (!encode_rows_map(&mq, p.dtype, p.q, D, p.geom.g, p.geom.tpt) ||
      !encode_keys_map(&mk, p.dtype, p.k, D, p.geom.box_rows) ||
      !encode_keys_map(&mv, p.dtype, p.v, D, p.geom.box_rows))
    return GPO_BAD_ARGS;
  FwdArgs a;
  a.geom = p.geom;
  a.out = p.out;
  a.lse = p.lse;
  a.o_batch = p.o_batch;
  a.o_token = p.o_token;
  a.o_head = p.o_head;
  a.scale_log2 = p.scale * 1.4426950408889634f;
  a.err = c.err;
  const int64_t items = static_cast<int64_t>(p.geom.tiles) * p.geom.batch * p.geom.heads_kv;
  if (items > (1ll << 31) - 1024) return GPO_BAD_ARGS;
  a.items = static_cast<int>(items);
  auto kern = attn_fwd_kernel<T, FMT, D, PAGED>;
  constexpr uint32_t dyn = (128u + 2u * kFwdStages * kOpsBN) * D * 2u + 1024u;
  gpo_status s = ensure_smem_attr(reinterpret_cast<const void*>(kern), dyn);
  if (s != GPO_OK) return s;
  const unsigned grid = static_cast<unsigned>(
      std::min<int64_t>(items, c.sm_count > 0 ? c.sm_count : 148));
  kern<<<grid, kFwdThreads, dyn, c.stream>>>(mq, mk, mv, a);
  return launch_status();
}

template <bool PAGED>
static gpo_status run_fwd_type(const AttnProblem& p, const LaunchCtx& c) {
  if (p.dtype == GPO_BFLOAT16)
    return p.dim == 128 ? run_fwd<__nv_bfloat16, 1, 128, PAGED>(p, c)
                        : run_fwd<__nv_bfloat16, 1, 64, PAGED>(p, c);
  return p.dim == 128 ? run_fwd<__half, 0, 128, PAGED>(p, c)
                      : run_fwd<__half, 0, 64, PAGED>(p, c);
}

gpo_status launch_attn_forward(const AttnProblem& p, const LaunchCtx& c) {
  return p.paged ? run_fwd_type<true>(p, c) : run_fwd_type<false>(p, c);
}

}  // namespace gpo
