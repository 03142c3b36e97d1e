// C entry points of the window / paged attention operators (include/gpo.h):
// argument checks, then the launchers of attn_fwd_ops.cu, attn_grad_ops.cu
// and cache_ops.cu.
#include <cmath>
#include <string>

#include "attn_ops.cuh"

namespace gpo {

namespace {

// Collects the reason of the first refusal.
struct Refusal {
  gpo_status status = GPO_OK;
  std::string why;
  bool no(gpo_status s, const std::string& w) {
    if (status == GPO_OK) {
      status = s;
      why = w;
    }
    return false;
  }
};

bool check_common(int dtype, int dim, int hq, int hk, int64_t window, int64_t sinks, float scale,
                  Refusal& r) {
  if (dtype != GPO_FLOAT16 && dtype != GPO_BFLOAT16)
    return r.no(GPO_BAD_CONFIG, "dtype must be float16 or bfloat16");
  if (dim != 64 && dim != 128)
    return r.no(GPO_BAD_CONFIG, "head_dim must be 64 or 128, got " + std::to_string(dim));
  if (hk < 1 || hq < 1 || hq % hk != 0)
    return r.no(GPO_BAD_ARGS, "heads_q (" + std::to_string(hq) + ") must be a multiple of heads_kv (" +
                                  std::to_string(hk) + ")");
  if (hq / hk > 128)
    return r.no(GPO_BAD_CONFIG, "at most 128 query heads per kv head");
  if (window < 0 || sinks < 0) return r.no(GPO_BAD_ARGS, "window and sinks must not be negative");
  // beyond, scale * log2(e) leaves the normal numbers and may meet a masked
  // score as 0 * -inf
  if (scale != 0.f && !(scale >= 0x1p-126f && scale <= 0x1p126f))
    return r.no(GPO_BAD_ARGS, "scale must be positive and finite, in [2^-126, 2^126]");
  return true;
}

// One strided tensor; `batch`, `tokens`: how far its strides are stepped.
bool check_heads(const gpo_heads& t, const char* name, int64_t batch, int64_t tokens, int heads,
                 Refusal& r) {
  if (!t.ptr) return r.no(GPO_BAD_ARGS, std::string(name) + " is null");
  if (!aligned16(t.ptr)) return r.no(GPO_BAD_ARGS, std::string(name) + " is not 16-byte aligned");
  const int64_t n[3] = {batch, tokens, heads};
  const int64_t s[3] = {t.stride_batch, t.stride_token, t.stride_head};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (s[i] < 0 || s[i] % 8 != 0 || s[i] >= (1ll << 38)))
      return r.no(GPO_BAD_ARGS, std::string(name) +
                                    ": strides must be multiples of 8 elements, 0 <= stride < 2^38");
  return true;
}

// An array of 32-bit values (null is the caller's matter).
bool check_array(const void* p, const char* name, Refusal& r) {
  if (reinterpret_cast<uintptr_t>(p) & 3u)
    return r.no(GPO_BAD_ARGS, std::string(name) + " is not 4-byte aligned");
  return true;
}

// Strides an output must not fold onto itself.
bool check_written(const gpo_heads& t, const char* name, int64_t batch, int64_t tokens, int heads,
                   int dim, Refusal& r) {
  if (!check_heads(t, name, batch, tokens, heads, r)) return false;
  const int64_t n[3] = {batch, tokens, heads};
  const int64_t s[3] = {t.stride_batch, t.stride_token, t.stride_head};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && s[i] < dim)
      return r.no(GPO_BAD_ARGS, std::string(name) + ": written rows overlap");
  return true;
}

int clamp_len(int64_t v) { return v > kOpsNoWindow ? kOpsNoWindow : static_cast<int>(v); }

void set_mask(AttnGeom& g, int64_t window, int64_t sinks, int64_t most_keys) {
  g.window = window == 0 || window >= most_keys ? kOpsNoWindow : static_cast<int>(window);
  // without a window every key a sink could add is visible already
  g.sinks = g.window == kOpsNoWindow ? 0 : clamp_len(sinks < most_keys ? sinks : most_keys);
}

HeadsView view(const gpo_heads& t, int64_t batch, int64_t tokens, int64_t heads) {
  return HeadsView{t.ptr, batch, tokens, heads, t.stride_batch, t.stride_token, t.stride_head};
}

// Sizes, types and mask of a dense problem; its pointers only where asked.
bool dense_problem(const gpo_window_args& a, bool pointers, AttnProblem& p, Refusal& r) {
  if (!check_common(a.dtype, a.head_dim, a.heads_q, a.heads_kv, a.window, a.sinks, a.scale, r))
    return false;
  if (a.batch < 0 || a.q_len < 0 || a.kv_len < 0 || a.batch > 65535 || a.q_len > kOpsMaxLen ||
      a.kv_len > kOpsMaxLen)
    return r.no(GPO_BAD_ARGS, "batch must be in [0, 65535], lengths in [0, 2^30]");
  if (a.reserved != 0) return r.no(GPO_BAD_ARGS, "reserved must be 0");
  AttnGeom& g = p.geom;
  g = AttnGeom{};
  g.batch = static_cast<int>(a.batch);
  g.q_len = static_cast<int>(a.q_len);
  g.kv_len = static_cast<int>(a.kv_len);
  g.heads_kv = a.heads_kv;
  g.g = a.heads_q / a.heads_kv;
  g.tpt = 128 / g.g;
  g.tiles = static_cast<int>(cdiv(static_cast<uint64_t>(a.q_len), static_cast<uint64_t>(g.tpt)));
  g.box_rows = kOpsBN;
  set_mask(g, a.window, a.sinks, a.kv_len);
  p.dtype = a.dtype;
  p.dim = a.head_dim;
  p.paged = false;
  p.scale = a.scale != 0.f ? a.scale : 1.0f / std::sqrt(static_cast<float>(a.head_dim));
  if (!pointers || a.batch == 0 || a.q_len == 0) return true;
  if (!check_heads(a.q, "q", a.batch, a.q_len, a.heads_q, r)) return false;
  p.q = view(a.q, a.batch, a.q_len, a.heads_q);
  if (a.kv_len > 0) {
    if (!check_heads(a.k, "k", a.batch, a.kv_len, a.heads_kv, r) ||
        !check_heads(a.v, "v", a.batch, a.kv_len, a.heads_kv, r))
      return false;
    p.k = view(a.k, a.batch, a.kv_len, a.heads_kv);
    p.v = view(a.v, a.batch, a.kv_len, a.heads_kv);
  } else {
    // no block is loaded, but a tensor map describes at least one row
    p.k = p.v = view(a.q, 1, 1, a.heads_kv);
  }
  return true;
}

gpo_status refuse(const Refusal& r, char* log, size_t cap) {
  write_log(log, cap, r.why);
  return r.status;
}

bool paged_problem(const gpo_paged_args& a, bool pointers, bool attention, AttnProblem& p,
                   Refusal& r) {
  if (!check_common(a.dtype, a.head_dim, a.heads_q, a.heads_kv, a.window, a.sinks, a.scale, r))
    return false;
  if (a.reserved != 0) return r.no(GPO_BAD_ARGS, "reserved must be 0");
  if (a.num_seqs < 0 || a.num_seqs > 65535 || a.tokens < 0 || a.tokens > kOpsMaxLen ||
      a.max_q < 0 || a.max_q > kOpsMaxLen)
    return r.no(GPO_BAD_ARGS, "num_seqs must be in [0, 65535], tokens and max_q in [0, 2^30]");
  if (a.page_size < 8 || a.page_size % 8 != 0 || a.page_size > (1 << 16))
    return r.no(GPO_BAD_CONFIG, "page_size must be a multiple of 8 in [8, 65536], got " +
                                    std::to_string(a.page_size));
  if (a.num_pages < 0 || a.num_pages > kOpsMaxLen || a.table_width < 0 ||
      a.table_width * a.page_size > kOpsMaxLen)
    return r.no(GPO_BAD_ARGS, "num_pages and table_width * page_size must be in [0, 2^30]");
  if (a.num_seqs > 1 && a.table_stride < a.table_width)
    return r.no(GPO_BAD_ARGS, "table_stride is less than table_width");
  AttnGeom& g = p.geom;
  g = AttnGeom{};
  g.q_start = a.q_start;
  g.kv_lens = a.kv_len;
  g.table = a.page_table;
  g.table_stride = a.table_stride;
  g.table_width = static_cast<int>(a.table_width);
  g.page_size = static_cast<int>(a.page_size);
  g.box_rows = 8;
  while (g.box_rows < kOpsBN && a.page_size % (2 * g.box_rows) == 0) g.box_rows *= 2;
  g.num_pages = static_cast<int>(a.num_pages);
  g.batch = static_cast<int>(a.num_seqs);
  g.q_len = static_cast<int>(a.max_q < a.tokens ? a.max_q : a.tokens);
  g.tokens = static_cast<int>(a.tokens);
  g.heads_kv = a.heads_kv;
  g.g = a.heads_q / a.heads_kv;
  g.tpt = 128 / g.g;
  g.tiles = static_cast<int>(cdiv(static_cast<uint64_t>(g.q_len), static_cast<uint64_t>(g.tpt)));
  set_mask(g, a.window, a.sinks, a.table_width * a.page_size);
  p.dtype = a.dtype;
  p.dim = a.head_dim;
  p.paged = true;
  p.scale = a.scale != 0.f ? a.scale : 1.0f / std::sqrt(static_cast<float>(a.head_dim));
  if (!pointers || a.num_seqs == 0 || a.tokens == 0) return true;
  if (!a.q_start || !a.kv_len || (a.table_width > 0 && !a.page_table))
    return r.no(GPO_BAD_ARGS, "page_table, q_start or kv_len is null");
  if (!check_array(a.page_table, "page_table", r) || !check_array(a.q_start, "q_start", r) ||
      !check_array(a.kv_len, "kv_len", r) || !check_array(a.lse, "lse", r))
    return false;
  if (a.num_pages > 0) {
    for (int i = 0; i < 2; ++i) {
      const gpo_heads& t = i ? a.v_pages : a.k_pages;
      const char* name = i ? "v_pages" : "k_pages";
      if (attention ? !check_heads(t, name, a.num_pages, a.page_size, a.heads_kv, r)
                    : !check_written(t, name, a.num_pages, a.page_size, a.heads_kv, a.head_dim, r))
        return false;
    }
    p.k = view(a.k_pages, a.num_pages, a.page_size, a.heads_kv);
    p.v = view(a.v_pages, a.num_pages, a.page_size, a.heads_kv);
  }
  if (attention) {
    if (!check_heads(a.q, "q", 1, a.tokens, a.heads_q, r) ||
        !check_written(a.out, "out", 1, a.tokens, a.heads_q, a.head_dim, r))
      return false;
    p.q = view(a.q, 1, a.tokens, a.heads_q);
    if (a.num_pages == 0) p.k = p.v = view(a.q, 1, 1, a.heads_kv);
    p.out = a.out.ptr;
    p.o_batch = 0;
    p.o_token = a.out.stride_token;
    p.o_head = a.out.stride_head;
    p.lse = a.lse;
  } else {
    if (!check_heads(a.k_new, "k_new", 1, a.tokens, a.heads_kv, r) ||
        !check_heads(a.v_new, "v_new", 1, a.tokens, a.heads_kv, r))
      return false;
    p.k_new = view(a.k_new, 1, a.tokens, a.heads_kv);
    p.v_new = view(a.v_new, 1, a.tokens, a.heads_kv);
  }
  return true;
}

// Runs `launch` with the current device's context; nothing throws past it.
template <typename F>
gpo_status guarded(void* stream, char* log, size_t cap, F&& launch) {
  LaunchCtx ctx;
  gpo_status s = launch_ctx(stream, &ctx);
  if (s == GPO_OK) s = launch(ctx);
  if (s != GPO_OK) write_log(log, cap, std::string(gpo_status_name(s)) + " at launch");
  return s;
}

}  // namespace

}  // namespace gpo

using namespace gpo;

extern "C" {

gpo_status gpo_window_attention(const gpo_window_args* a, void* stream, char* log, size_t cap) {
  if (!a) return GPO_BAD_ARGS;
  try {
    write_log(log, cap, "");
    AttnProblem p{};
    Refusal r;
    if (!dense_problem(*a, true, p, r)) return refuse(r, log, cap);
    if (a->batch == 0 || a->q_len == 0) return GPO_OK;
    if (!check_written(a->out, "out", a->batch, a->q_len, a->heads_q, a->head_dim, r) ||
        !check_array(a->lse, "lse", r))
      return refuse(r, log, cap);
    p.out = a->out.ptr;
    p.o_batch = a->out.stride_batch;
    p.o_token = a->out.stride_token;
    p.o_head = a->out.stride_head;
    p.lse = a->lse;
    return guarded(stream, log, cap, [&](LaunchCtx& c) { return launch_attn_forward(p, c); });
  } catch (...) {
    return GPO_INTERNAL;
  }
}

gpo_status gpo_window_kernel(const gpo_window_args* a, char* name, size_t cap) {
  if (!a) return GPO_BAD_ARGS;
  try {
    AttnProblem p{};
    Refusal r;
    if (!dense_problem(*a, false, p, r)) return refuse(r, name, cap);
    write_log(name, cap, attn_forward_name(p));
    return GPO_OK;
  } catch (...) {
    return GPO_INTERNAL;
  }
}

gpo_status gpo_window_workspace(const gpo_window_args* a, uint64_t* bytes, char* log,
                                size_t cap) {
  if (!a || !bytes) return GPO_BAD_ARGS;
  try {
    write_log(log, cap, "");
    *bytes = 0;
    AttnProblem p{};
    Refusal r;
    if (!dense_problem(*a, false, p, r)) return refuse(r, log, cap);
    *bytes = attn_grad_workspace(p);
    return GPO_OK;
  } catch (...) {
    return GPO_INTERNAL;
  }
}

gpo_status gpo_window_attention_grad(const gpo_window_args* a, void* stream, char* log,
                                     size_t cap) {
  if (!a) return GPO_BAD_ARGS;
  try {
    write_log(log, cap, "");
    AttnProblem p{};
    Refusal r;
    if (!dense_problem(*a, true, p, r)) return refuse(r, log, cap);
    if (a->batch == 0 || (a->q_len == 0 && a->kv_len == 0)) return GPO_OK;
    AttnGradProblem gp{};
    const int64_t b = a->batch, q = a->q_len, n = a->kv_len;
    if (q > 0) {
      if (!check_heads(a->out, "out", b, q, a->heads_q, r) ||
          !check_heads(a->dout, "dout", b, q, a->heads_q, r) ||
          !check_written(a->dq, "dq", b, q, a->heads_q, a->head_dim, r) ||
          !check_array(a->lse, "lse", r))
        return refuse(r, log, cap);
      if (!a->lse) {
        r.no(GPO_BAD_ARGS, "lse is null");
        return refuse(r, log, cap);
      }
    }
    if (n > 0 && (!check_written(a->dk, "dk", b, n, a->heads_kv, a->head_dim, r) ||
                  !check_written(a->dv, "dv", b, n, a->heads_kv, a->head_dim, r)))
      return refuse(r, log, cap);
    if (q == 0 && n > 0) {
      // no query: dk and dv are 0, and the maps describe one row of k
      if (!check_heads(a->k, "k", b, n, a->heads_kv, r) ||
          !check_heads(a->v, "v", b, n, a->heads_kv, r))
        return refuse(r, log, cap);
      p.k = view(a->k, b, n, a->heads_kv);
      p.v = view(a->v, b, n, a->heads_kv);
      p.q = gp.dout = HeadsView{a->k.ptr, 1, 1, a->heads_q, 0, 0, a->head_dim};
    } else {
      gp.dout = view(a->dout, b, q, a->heads_q);
    }
    gp.out = view(a->out, b, q, a->heads_q);
    gp.dq = view(a->dq, b, q, a->heads_q);
    gp.dk = view(a->dk, b, n, a->heads_kv);
    gp.dv = view(a->dv, b, n, a->heads_kv);
    gp.lse = a->lse;
    gp.workspace = a->workspace;
    const uint64_t need = attn_grad_workspace(p);
    if (need > 0 && (!a->workspace || a->workspace_bytes < need ||
                     (reinterpret_cast<uintptr_t>(a->workspace) & 255u))) {
      r.no(GPO_BAD_ARGS, "workspace must be 256-byte aligned and hold " + std::to_string(need) +
                             " bytes, got " + std::to_string(a->workspace_bytes));
      return refuse(r, log, cap);
    }
    return guarded(stream, log, cap, [&](LaunchCtx& c) { return launch_attn_grad(p, gp, c); });
  } catch (...) {
    return GPO_INTERNAL;
  }
}

gpo_status gpo_paged_kernel(const gpo_paged_args* a, char* name, size_t cap) {
  if (!a) return GPO_BAD_ARGS;
  try {
    AttnProblem p{};
    Refusal r;
    if (!paged_problem(*a, false, true, p, r)) return refuse(r, name, cap);
    write_log(name, cap, attn_forward_name(p));
    return GPO_OK;
  } catch (...) {
    return GPO_INTERNAL;
  }
}

gpo_status gpo_paged_workspace(const gpo_paged_args* a, uint64_t* bytes, char* log, size_t cap) {
  if (!a || !bytes) return GPO_BAD_ARGS;
  try {
    write_log(log, cap, "");
    *bytes = 0;
    AttnProblem p{};
    Refusal r;
    if (!paged_problem(*a, false, false, p, r)) return refuse(r, log, cap);
    *bytes = attn_paged_workspace(p);
    return GPO_OK;
  } catch (...) {
    return GPO_INTERNAL;
  }
}

gpo_status gpo_paged_attention(const gpo_paged_args* a, void* stream, char* log, size_t cap) {
  if (!a) return GPO_BAD_ARGS;
  try {
    write_log(log, cap, "");
    AttnProblem p{};
    Refusal r;
    if (!paged_problem(*a, true, true, p, r)) return refuse(r, log, cap);
    if (a->num_seqs == 0 || a->tokens == 0 || p.geom.q_len == 0) return GPO_OK;
    const uint64_t need = attn_paged_workspace(p);
    if (!a->workspace || a->workspace_bytes < need ||
        (reinterpret_cast<uintptr_t>(a->workspace) & 255u)) {
      r.no(GPO_BAD_ARGS, "workspace must be 256-byte aligned and hold " + std::to_string(need) +
                             " bytes, got " + std::to_string(a->workspace_bytes));
      return refuse(r, log, cap);
    }
    p.workspace = a->workspace;
    return guarded(stream, log, cap, [&](LaunchCtx& c) { return launch_attn_forward(p, c); });
  } catch (...) {
    return GPO_INTERNAL;
  }
}

gpo_status gpo_cache_append(const gpo_paged_args* a, void* stream, char* log, size_t cap) {
  if (!a) return GPO_BAD_ARGS;
  try {
    write_log(log, cap, "");
    AttnProblem p{};
    Refusal r;
    if (!paged_problem(*a, true, false, p, r)) return refuse(r, log, cap);
    if (a->num_seqs == 0 || a->tokens == 0 || a->num_pages == 0) return GPO_OK;
    return guarded(stream, log, cap, [&](LaunchCtx& c) { return launch_cache_append(p, c); });
  } catch (...) {
    return GPO_INTERNAL;
  }
}

}  // extern "C"
