// Append of new tokens' K/V rows to a paged cache: a copy with a gather of
// addresses.  Its floor is the rows' bytes, read and written once; for a
// few tokens a launch.  One thread moves one 16-byte vector of a row of K
// and of V; the token's sequence is found by a binary search of q_start,
// whose values every thread of a block reads from the same cache lines.
// 8 chunks of up to 1024 tokens (8 heads, D 128, 16 bits; 57 MB): 11.7 us, 4.8
// TB/s, of which some 4 us are the launch and the chain of loads before the
// copy; 64 single tokens: 3.9 us.  Two vectors per thread were slower (3.1 ->
// 3.5 us without the launch, 64 tokens).
#include "attn_ops.cuh"

namespace gpo {

struct AppendArgs {
  AttnGeom geom;
  const uint4 *k_new, *v_new;
  uint4 *k_pages, *v_pages;
  // in 16-byte vectors
  int64_t kn_token, kn_head, vn_token, vn_head;
  int64_t kp_page, kp_slot, kp_head, vp_page, vp_slot, vp_head;
  int vecs;  // vectors of a row
  unsigned int* err;
};

// One vector of a token's K and V.
__device__ __forceinline__ void append_vector(const AppendArgs& a) {
  const AttnGeom& g = a.geom;
  const int per_token = g.heads_kv * a.vecs;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t t64 = i / per_token;
  if (t64 >= g.tokens) return;
  const int t = static_cast<int>(t64);
  const int e = static_cast<int>(i - t64 * per_token);
  const int h = e / a.vecs, x = e % a.vecs;
  // the sequence b with q_start[b] <= t < q_start[b + 1]
  int lo = 0, hi = g.batch;
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (__ldg(g.q_start + m) <= t)
      lo = m;
    else
      hi = m;
  }
  const int first = __ldg(g.q_start + lo), end = __ldg(g.q_start + lo + 1);
  const int keys = __ldg(g.kv_lens + lo);
  // a sequence that does not fit (attn_seq) is not written, not even in part
  if (t < first || t >= end || first < 0 || end > g.tokens ||
      keys > g.table_width * g.page_size)
    return;
  const int slot = keys - (end - t);
  if (slot < 0) return;  // a token in front of the first key has none
  const int at = slot / g.page_size;
  const int page = __ldg(g.table + lo * g.table_stride + at);
  if (page < 0 || page >= g.num_pages) return;
  const int row = slot - at * g.page_size;
  const uint4 kv = __ldcs(a.k_new + t * a.kn_token + h * a.kn_head + x);
  const uint4 vv = __ldcs(a.v_new + t * a.vn_token + h * a.vn_head + x);
  a.k_pages[page * a.kp_page + row * a.kp_slot + h * a.kp_head + x] = kv;
  a.v_pages[page * a.vp_page + row * a.vp_slot + h * a.vp_head + x] = vv;
}

__global__ void __launch_bounds__(256) cache_append_kernel(const AppendArgs a) {
  const AttnGeom& g = a.geom;
  let_next_start();
  wait_for_previous();
  append_vector(a);
  // sequences that do not fit are reported, those that no token leads to included
  if (blockIdx.x == 0)
    for (int b = threadIdx.x; b < g.batch; b += 256) attn_seq<true>(g, b, a.err);
}

gpo_status launch_cache_append(const AttnProblem& p, const LaunchCtx& c) {
  AppendArgs a;
  a.geom = p.geom;
  a.k_new = static_cast<const uint4*>(p.k_new.ptr);
  a.v_new = static_cast<const uint4*>(p.v_new.ptr);
  a.k_pages = static_cast<uint4*>(const_cast<void*>(p.k.ptr));
  a.v_pages = static_cast<uint4*>(const_cast<void*>(p.v.ptr));
  a.kn_token = p.k_new.s_token / 8;
  a.kn_head = p.k_new.s_head / 8;
  a.vn_token = p.v_new.s_token / 8;
  a.vn_head = p.v_new.s_head / 8;
  a.kp_page = p.k.s_batch / 8;
  a.kp_slot = p.k.s_token / 8;
  a.kp_head = p.k.s_head / 8;
  a.vp_page = p.v.s_batch / 8;
  a.vp_slot = p.v.s_token / 8;
  a.vp_head = p.v.s_head / 8;
  a.vecs = p.dim / 8;
  a.err = c.err;
  a.geom.q_len = a.geom.tokens;  // max_q bounds the attention's tiles, not a copy
  const uint64_t n = static_cast<uint64_t>(p.geom.tokens) * p.geom.heads_kv * a.vecs;
  const uint64_t blocks = cdiv(n, 256);
  if (blocks > 0x7fffffffull) return GPO_BAD_ARGS;
  return launch_in_order(cache_append_kernel, static_cast<unsigned>(blocks), 256, 0, c.stream, a);
}

}  // namespace gpo
