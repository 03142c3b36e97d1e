// What the window / paged attention kernels share: which keys a tile of
// query rows sees, tensor maps over strided heads, and the launch records.
//
// Heads are grouped: query head h reads kv head h / g.  A tile of query rows
// packs all g query heads of one kv head: row r of a tile that starts at
// token t0 is token t0 + r / g, head r % g, so one K/V block serves g heads
// from a single shared-memory copy.  A tile holds tpt = 128 / g whole tokens
// (rows tpt * g .. 127 are unused when g does not divide 128).
//
// Mask: token i of a sequence with q_len new tokens and kv_len keys stands
// at p = i + kv_len - q_len and sees key j iff j <= p and
// (p - j < window or j < sinks).
#pragma once

#include <string>

#include "gpo_common.cuh"
#include "gpo_internal.h"

namespace gpo {

constexpr int kOpsBN = 128;              // keys per block
constexpr int kOpsNoWindow = 1 << 30;    // a window that reaches every key
constexpr int kOpsMaxLen = 1 << 30;      // largest q_len / kv_len

// The part of a problem that every role of a kernel needs.
struct AttnGeom {
  const int* q_start;   // paged: first row of each sequence (batch + 1 values)
  const int* kv_lens;   // paged: keys of each sequence, its new tokens included
  const int* table;     // paged: page of every page_size slots
  int64_t table_stride;
  int table_width;
  int page_size, box_rows, num_pages;
  int batch, q_len, kv_len;  // q_len: dense length, or the most a sequence has
  int tokens;                // paged: rows of q
  int heads_kv, g, tpt;
  int tiles;                 // dense: query tiles per sequence
  int window, sinks;
};

struct AttnSeq {
  int q_len, kv_len;
  int row0;  // first row of the sequence in the packed q (paged), else 0
  int off;   // position of token 0
};

// Lengths of sequence b.  Paged lengths are device data that the host has
// not seen: values that do not fit the buffers are cut to what does.
template <bool PAGED>
__device__ __forceinline__ AttnSeq attn_seq(const AttnGeom& g, int b, unsigned int* err) {
  AttnSeq s;
  if constexpr (PAGED) {
    const int a = __ldg(g.q_start + b), e = __ldg(g.q_start + b + 1);
    const int n = __ldg(g.kv_lens + b);
    const int64_t cap = static_cast<int64_t>(g.table_width) * g.page_size;
    s.row0 = a;
    s.q_len = e - a;
    s.kv_len = n;
    if (a < 0 || e < a || e > g.tokens || s.q_len > g.q_len || n < 0 || n > cap) {
      s.row0 = 0;
      s.q_len = 0;
      s.kv_len = 0;
      atomicOr(err, kErrBadLaunch);
    }
  } else {
    s.row0 = 0;
    s.q_len = g.q_len;
    s.kv_len = g.kv_len;
  }
  s.off = s.kv_len - s.q_len;
  return s;
}

// K/V blocks that some row of tokens [t0, t1) sees: the sink blocks
// [0, sink_blocks) and then the blocks first, first + 1, ... of the window.
struct AttnBlocks {
  int n, sink_blocks, first;
  __device__ __forceinline__ int at(int i) const {
    return i < sink_blocks ? i : first + i - sink_blocks;
  }
};

__device__ __forceinline__ AttnBlocks attn_blocks(const AttnGeom& g, const AttnSeq& s, int t0,
                                                  int t1) {
  AttnBlocks b{0, 0, 0};
  const int hi = t1 - 1 + s.off;  // last position: the last key any row sees
  if (t0 >= t1 || hi < 0) return b;
  const int lo = max(0, t0 + s.off - g.window + 1);
  b.first = lo / kOpsBN;
  b.sink_blocks = min(b.first, (min(g.sinks, hi + 1) + kOpsBN - 1) / kOpsBN);
  b.n = b.sink_blocks + hi / kOpsBN - b.first + 1;
  return b;
}

// Keys [sinks, attn_unseen) are in front of every token's window.
__device__ __forceinline__ int attn_unseen(const AttnGeom& g, const AttnSeq& s) {
  return max(0, s.off - g.window + 1);
}
// What a key holds that no token of its sequence sees must not reach a sum:
// its weight is 0, but 0 * NaN is not.  Boxes (box_rows keys, the unit of a
// copy) of such keys alone are not copied; the others are cleared in shared
// memory.  Dense blocks are one box, and none without a visible key is loaded.
__device__ __forceinline__ bool attn_box_unseen(const AttnGeom& g, const AttnSeq& s, int key) {
  return key >= g.sinks && key + g.box_rows <= attn_unseen(g, s);
}
// Rows of the block at key0 to clear, [a0, a1) behind the sinks and [b0, b1)
// in front of the window (either may be empty, both may overlap).
struct AttnUnseenRows {
  int a0, a1, b0, b1;
  __device__ __forceinline__ bool any() const { return a0 < a1 || b0 < b1; }
};
__device__ __forceinline__ AttnUnseenRows attn_unseen_rows(const AttnGeom& g, const AttnSeq& s,
                                                           int key0) {
  const int a = max(key0, g.sinks), b = min(key0 + kOpsBN, attn_unseen(g, s));
  const int box = g.box_rows - 1;
  return AttnUnseenRows{a - key0, min(b, (a + box) & ~box) - key0, max(a, b & ~box) - key0,
                        b - key0};
}

// Bits [a, b) of word c of a 32-bit mask row (bit i of word c is index 32c + i).
__device__ __forceinline__ uint32_t bits_below(int n, int c) {
  const int k = n - 32 * c;
  return k <= 0 ? 0u : k >= 32 ? 0xffffffffu : (1u << k) - 1u;
}

// Mask of a packed 16-bit pair: 0xffff in each half whose bit (2 i, 2 i + 1)
// of `see` is set.  The bit is shifted to the top of its byte and replicated
// from there by the byte permutation's sign mode; the eight shifts are shared
// by the 16 pairs of a word.
__device__ __forceinline__ uint32_t pair_mask(uint32_t see, int i) {
  const int lo = 2 * i, hi = 2 * i + 1;
  const uint32_t a = see << (7 - (lo & 7)), b = see << (7 - (hi & 7));
  const uint32_t from_a = 8u | static_cast<uint32_t>(lo >> 3);
  const uint32_t from_b = 8u | 4u | static_cast<uint32_t>(hi >> 3);
  uint32_t m;
  asm("prmt.b32 %0, %1, %2, %3;"
      : "=r"(m)
      : "r"(a), "r"(b), "r"(from_a | from_a << 4 | from_b << 8 | from_b << 12));
  return m;
}

// Keys of a block that a row at position p sees: i <= p - key0 and
// (i > p - key0 - window or i < sinks - key0), i counted from the block's
// first key; as mask words, which cost a test and a select per score.
struct RowMask {
  int end, lo, sink;
  __device__ __forceinline__ uint32_t word(int c) const {
    return bits_below(end, c) & (~bits_below(lo, c) | bits_below(sink, c));
  }
};

__device__ __forceinline__ RowMask row_mask(const AttnGeom& g, int p, int key0) {
  return RowMask{p - key0 + 1, p - g.window + 1 - key0, g.sinks - key0};
}

// Whether some row of tokens [t0, t1) misses a key of the block.
__device__ __forceinline__ bool block_is_masked(const AttnGeom& g, const AttnSeq& s, int t0,
                                                int t1, int key0) {
  return key0 + kOpsBN - 1 > t0 + s.off || (t1 - 1 + s.off - g.window + 1 > key0 &&
                                            key0 + kOpsBN > g.sinks);
}

// 2^x of two values on the FMA pipe: x = n + f with f in [-1/2, 1/2], 2^f by
// a polynomial of least relative error on that interval (7.5e-5 of degree 3,
// 2.6e-6 of degree 4; fitted by iteratively reweighted least squares), 2^n
// multiplied in.  For P of the gradient (degree 3: bfloat16, 4: float16), which
// reaches its sums rounded to 16 bits, by itself or as the factor of dS = P *
// (dP - delta): dS takes over P's relative error, a 52nd (a 188th) of what its
// own rounding may take.  x below -126 gives 2^-126, NaN stays NaN.
template <int DEGREE>
__device__ __forceinline__ float2 exp2_fma(float2 x) {
  constexpr float kRound = 12582912.f;  // 1.5 * 2^23: adding it rounds to integer
  auto both = [](float v) { return make_float2(v, v); };
  asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(x.x));  // -126
  asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(x.y));
  const float2 n = __fadd2_rn(x, both(kRound));
  const float2 f = __fadd2_rn(x, __ffma2_rn(n, both(-1.f), both(kRound)));
  float2 p;
  if constexpr (DEGREE == 3) {
    p = __ffma2_rn(f, both(0.05517167f), both(0.24261113f));
    p = __ffma2_rn(f, p, both(0.69326097f));
    p = __ffma2_rn(f, p, both(0.99992806f));
  } else {
    p = __ffma2_rn(f, both(0.009570102f), both(0.05591786f));
    p = __ffma2_rn(f, p, both(0.24024744f));
    p = __ffma2_rn(f, p, both(0.6931218f));
    p = __ffma2_rn(f, p, both(0.9999993f));
  }
  // the integer n sits in the low bits of n + kRound
  return __fmul2_rn(p, make_float2(__uint_as_float((__float_as_uint(n.x) << 23) + 0x3F800000u),
                                   __uint_as_float((__float_as_uint(n.y) << 23) + 0x3F800000u)));
}

// Eight 16-bit pairs to global memory: one 32-byte store where the address
// allows (a row per lane: a whole sector per lane and half the wavefronts).
// Gradients of 8192 tokens whose rows start on 32 bytes against 16: 447..460
// us and 452..465.
__device__ __forceinline__ void store_pairs8(void* dst, const uint32_t* v, bool wide) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(dst)[0] = make_uint4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<uint4*>(dst)[1] = make_uint4(v[4], v[5], v[6], v[7]);
  }
}

// True in one thread of a converged warp.  Single-thread roles branch on this
// and not on the lane index: the compiler then knows that one thread runs
// and keeps descriptors in uniform registers.  Measured: 38 cycles to issue
// an MMA and 32 a commit, 70 and 110 behind `lane == 0`, where an MMA
// executes in 64.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.u32 %0, 1, 0, P;\n\t}"
               : "=r"(p));
  return p != 0;
}

// A CTA of these kernels asks for all of its SM's TMEM, and one that has
// started early (see below) keeps it while it waits for the kernel before: on
// an SM where that kernel's CTA had not got its own yet, both would wait for
// good.  They never share an SM, as each takes more than half of its shared
// memory (228 KB, 1 KB of every CTA reserved).
constexpr uint32_t kOpsAloneBytes = 113u * 1024u;  // a CTA's own, more than

// Launch order within a stream: a kernel launched by launch_in_order may
// start (barriers, TMEM, descriptors) while the kernel before it still runs,
// and touches global memory only behind wait_for_previous.
__device__ __forceinline__ void wait_for_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void let_next_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// 5-D tiled load (see tma_load_3d).
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                            int32_t x, int32_t y, int32_t z, int32_t u,
                                            int32_t v) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(u), "r"(v)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                            int32_t x, int32_t y, int32_t z, int32_t u) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(u)
      : "memory");
}

// 5-D tiled store of a swizzled tile in this CTA's shared memory.
__device__ __forceinline__ void tma_store_5d(const CUtensorMap* map, uint32_t src, int32_t x,
                                             int32_t y, int32_t z, int32_t u, int32_t v) {
  asm volatile(
      "cp.async.bulk.tensor.5d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4, %5, %6}], "
      "[%1];" ::"l"(reinterpret_cast<uint64_t>(map)),
      "r"(src), "r"(x), "r"(y), "r"(z), "r"(u), "r"(v)
      : "memory");
}
__device__ __forceinline__ void bulk_commit() {
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// This thread's stores have read their shared memory / are done.
__device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}
__device__ __forceinline__ void bulk_wait() {
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

// Eight 16-bit values (four pairs) of a row into a 128-byte-swizzled tile of
// 128 rows: 16-byte chunk `c` (of 8 per 64 dims) of `row`.
__device__ __forceinline__ void stage_chunk(uint32_t tile, int row, int c, const uint32_t* v) {
  const uint32_t at = tile + (c / 8) * 128 * 128 + row * 128 + (((c % 8) ^ (row & 7)) << 4);
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3])
               : "memory");
}

// ------------------------------------------------------------------- host
// One strided (batch, token, head, dim) tensor of 16-bit elements.
struct HeadsView {
  const void* ptr;
  int64_t batch, tokens, heads;
  int64_t s_batch, s_token, s_head;  // elements
};

// See wait_for_previous.  Measured: 1 to 2 us per launch in a row of them.
template <typename... K, typename... A>
inline gpo_status launch_in_order(void (*kernel)(K...), unsigned grid, unsigned block,
                                  uint32_t dyn_smem, cudaStream_t stream, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(block, 1, 1);
  cfg.dynamicSmemBytes = dyn_smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) {
    cudaGetLastError();
    return GPO_LAUNCH_ERROR;
  }
  return launch_status();
}

// Whether a dense problem has keys that no token sees (attn_unseen).  Its
// kernels are instances of their own: the tests of the blocks' positions in
// loops that never clear one took 153.4 in place of 150.5 us (prompt of 8192,
// W 1024) and 28.9 in place of 28.4 (3 x 333 tokens, forward and gradient).
// Clearing costs 91.9 -> 94.4 us forward and 246 -> 256 back for 4096 queries
// behind 4096 more keys, W 1024, 4 sinks, 32 heads over 8 of D 128.
inline bool attn_has_unseen(const AttnGeom& g) {
  const int64_t off = static_cast<int64_t>(g.kv_len) - g.q_len;
  return g.q_len > 0 && off - g.window + 1 > g.sinks;
}

// Whether every row of `t` starts on 32 bytes (see store_pairs8).
inline bool rows_on_32(const HeadsView& t) {
  return (reinterpret_cast<uintptr_t>(t.ptr) & 31u) == 0 && (t.batch <= 1 || t.s_batch % 16 == 0) &&
         (t.tokens <= 1 || t.s_token % 16 == 0) && (t.heads <= 1 || t.s_head % 16 == 0);
}

// Tile of a query-side tensor: {64 dims, g heads, 1 kv head, tpt tokens}.
bool encode_rows_map(CUtensorMap* map, int dtype, const HeadsView& t, int dim, int g, int tpt);
// Block of a key-side tensor: {64 dims, 1 head, rows, 1 batch or page}.
bool encode_keys_map(CUtensorMap* map, int dtype, const HeadsView& t, int dim, int rows);

// A checked problem, as the entry points hand it to the launchers.
struct AttnProblem {
  AttnGeom geom;
  int dtype, dim;
  bool paged;
  float scale;
  HeadsView q, k, v;         // paged: k and v are the pages
  HeadsView k_new, v_new;    // append
  void* out;
  int64_t o_batch, o_token, o_head;
  float* lse;
  void* workspace;  // paged
};

// What the gradient adds to a dense problem.
struct AttnGradProblem {
  HeadsView out, dout, dq, dk, dv;
  const float* lse;
  void* workspace;
};

uint64_t attn_grad_workspace(const AttnProblem& p);
gpo_status launch_attn_grad(const AttnProblem& p, const AttnGradProblem& gp, const LaunchCtx& c);
uint64_t attn_paged_workspace(const AttnProblem& p);
std::string attn_forward_name(const AttnProblem& p);
gpo_status launch_attn_forward(const AttnProblem& p, const LaunchCtx& c);
gpo_status launch_cache_append(const AttnProblem& p, const LaunchCtx& c);

}  // namespace gpo
