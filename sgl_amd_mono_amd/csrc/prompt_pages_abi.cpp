// The C entry points of a prompt's own attention and a drafted tree's: index queries, page
// scores, page selection, attention over pages. Argument checks, workspaces, launches; no state.
#include <cmath>

#include "prompt_abi.h"

namespace {

using namespace mono::prompt;

int need_counts(int32_t requests, int32_t pt_stride, int32_t n_pages) {
  if (requests < 0 || pt_stride < 0 || n_pages < 0)
    return refuse("requests, pt_stride and n_pages must not be negative, got %d, %d, %d", requests, pt_stride, n_pages);
  return MONO_OK;
}

int need_heads(int32_t heads) {
  if (heads < 1 || heads > MAX_HEADS) return refuse("heads must be in [1, %d], got %d", MAX_HEADS, heads);
  return MONO_OK;
}

int attention_shape(int64_t tokens, int32_t heads, int32_t picks) {
  if (int rc = need_rows(tokens, "tokens")) return rc;
  if (int rc = need_heads(heads)) return rc;
  if (picks < 0 || picks > MAX_COLUMNS) return refuse("picks must be in [0, %d], got %d", MAX_COLUMNS, picks);
  return MONO_OK;
}

int tree_shape(int64_t nodes, int32_t heads, int32_t pt_stride) {
  if (int rc = need_rows(nodes, "nodes")) return rc;
  if (int rc = need_heads(heads)) return rc;
  if (pt_stride < 0) return refuse("pt_stride must not be negative, got %d", pt_stride);
  return MONO_OK;
}

// The plan of a call over its workspace: parts where its pages are shared out.
size_t paged_space(void* ws, int pages, Paged& p) {
  Space sp{static_cast<char*>(ws)};
  paged_plan(p, pages);
  if (!p.parts) return 0;
  const size_t rows = (size_t)p.parts * p.heads;
  p.part = sp.take<float>(rows * LATENT);
  p.part_m = sp.take<float>(rows);
  p.part_l = sp.take<float>(rows);
  if (p.tasks) p.plan = sp.take<NodePlan>(p.tokens);
  return sp.off;
}

int64_t paged_workspace(int64_t tokens, int32_t heads, int pages, bool tree) {
  Paged p{};
  const int32_t some = 0;
  p.tokens = tokens, p.heads = heads, p.requests = 1, p.starts = tree ? &some : nullptr;
  mono::abi_ok();
  return tokens ? (int64_t)paged_space(nullptr, pages, p) : 0;
}

int run_paged(Paged& p, int pages, float scale, void* ws, int64_t ws_bytes, void* stream) {
  if (int rc = need(p.q, "q", 16)) return rc;
  if (p.requests && p.pt_stride)
    if (int rc = need(p.page_table, "page_table", 4)) return rc;
  if (p.n_pages)
    if (int rc = need(p.kv, "kv", 16)) return rc;
  if (p.kv_scale)
    if (int rc = need(p.kv_scale, "kv_scale", 16)) return rc;
  if (int rc = need(p.out, "out", 16)) return rc;
  p.scale_log2 = (float)(scale * 1.4426950408889634);
  if (!std::isfinite(p.scale_log2)) return refuse("softmax_scale must be finite, also times log2(e), got %g", (double)scale);
  if (const size_t bytes = paged_space(nullptr, pages, p)) {
    if (int rc = need_space(ws, ws_bytes, bytes)) return rc;
    paged_space(ws, pages, p);
  }
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (hipError_t e = paged_attention(p, st)) return launched(e, "the attention over pages");
  return launched(p.parts ? join_attention(p, st) : hipSuccess, "the join of the attention's parts");
}

}  // namespace

extern "C" int mono_prompt_query(const mono_prompt_query_args* args, void* stream) {
  if (!args) return refuse("mono_prompt_query: args is NULL");
  const mono_prompt_query_args& a = *args;
  if (int rc = need_rows(a.tokens, "tokens")) return rc;
  if (a.max_pos < 0) return refuse("max_pos must not be negative, got %d", a.max_pos);
  if (a.tokens == 0) return mono::abi_ok();
  if (a.max_pos == 0) return refuse("max_pos must be at least 1, got 0");
  if (int rc = need_stride(a.x_stride, INDEX_HEADS * INDEX, a.f32 ? 4 : 8, "x_stride")) return rc;
  if (int rc = need(a.x, "x", 16)) return rc;
  if (int rc = need(a.pos, "pos", 4)) return rc;
  if (int rc = need(a.rope_cos, "rope_cos", 16)) return rc;
  if (int rc = need(a.rope_sin, "rope_sin", 16)) return rc;
  if (int rc = need(a.iq, "iq", 16)) return rc;
  if (int rc = need(a.iqs, "iqs", 4)) return rc;
  return launched(index_query(a, static_cast<hipStream_t>(stream)), "the index queries");
}

extern "C" int mono_prompt_scores(const mono_prompt_scores_args* args, void* stream) {
  if (!args) return refuse("mono_prompt_scores: args is NULL");
  const mono_prompt_scores_args& a = *args;
  if (int rc = need_rows(a.tokens, "tokens")) return rc;
  if (int rc = need_counts(a.requests, a.pt_stride, a.n_pages)) return rc;
  if (a.columns < 0 || a.columns > MAX_COLUMNS) return refuse("columns must be in [0, %d], got %d", MAX_COLUMNS, a.columns);
  if (a.tokens == 0 || a.columns == 0) return mono::abi_ok();
  if (int rc = need(a.iq, "iq", 16)) return rc;
  if (int rc = need(a.iqs, "iqs", 4)) return rc;
  if (int rc = need(a.iw, "iw", 8)) return rc;
  if (int rc = need(a.req, "req", 4)) return rc;
  if (int rc = need(a.pos, "pos", 4)) return rc;
  if (a.requests && a.pt_stride)
    if (int rc = need(a.page_table, "page_table", 4)) return rc;
  if (a.n_pages) {
    if (int rc = need(a.ikv, "ikv", 16)) return rc;
    if (int rc = need(a.iks, "iks", 4)) return rc;
  }
  if (int rc = need(a.out, "out", 4)) return rc;
  return launched(page_scores(a, static_cast<hipStream_t>(stream)), "the page scores");
}

extern "C" int mono_prompt_select(const mono_prompt_select_args* args, void* stream) {
  if (!args) return refuse("mono_prompt_select: args is NULL");
  const mono_prompt_select_args& a = *args;
  if (int rc = need_rows(a.tokens, "tokens")) return rc;
  if (a.columns < 1 || a.columns > MAX_COLUMNS) return refuse("columns must be in [1, %d], got %d", MAX_COLUMNS, a.columns);
  if (a.picks < 1 || a.picks > MAX_COLUMNS) return refuse("picks must be in [1, %d], got %d", MAX_COLUMNS, a.picks);
  if (a.first < 0 || a.last < 0 || a.first > a.picks - a.last)
    return refuse("first and last must not be negative nor sum to more than picks, got %d and %d of %d", a.first, a.last, a.picks);
  if (a.tokens == 0) return mono::abi_ok();
  if (int rc = need_stride(a.stride, a.columns, 1, "stride")) return rc;
  if (int rc = need(a.scores, "scores", 4)) return rc;
  if (int rc = need(a.pos, "pos", 4)) return rc;
  if (int rc = need(a.pages, "pages", 4)) return rc;
  return launched(select_pages(a, static_cast<hipStream_t>(stream)), "the page selection");
}

extern "C" int64_t mono_prompt_attention_workspace(int64_t tokens, int32_t heads, int32_t picks) {
  if (attention_shape(tokens, heads, picks)) return -1;
  return paged_workspace(tokens, heads, picks, false);
}

extern "C" int mono_prompt_attention(const mono_prompt_attention_args* args, void* stream) {
  if (!args) return refuse("mono_prompt_attention: args is NULL");
  const mono_prompt_attention_args& a = *args;
  if (int rc = attention_shape(a.tokens, a.heads, a.picks)) return rc;
  if (int rc = need_counts(a.requests, a.pt_stride, a.n_pages)) return rc;
  if (a.tokens == 0) return mono::abi_ok();
  if (int rc = need(a.req, "req", 4)) return rc;
  if (int rc = need(a.pos, "pos", 4)) return rc;
  if (a.picks)
    if (int rc = need(a.pages, "pages", 4)) return rc;
  Paged p{};
  p.q = a.q, p.tokens = a.tokens, p.heads = a.heads;
  p.req = a.req, p.pos = a.pos, p.pages = a.pages, p.picks = a.picks;
  p.page_table = a.page_table, p.requests = a.requests, p.pt_stride = a.pt_stride, p.n_pages = a.n_pages;
  p.kv = a.kv, p.kv_scale = a.kv_scale, p.out = a.out;
  return run_paged(p, a.picks, a.softmax_scale, a.workspace, a.workspace_bytes, stream);
}

extern "C" int64_t mono_prompt_tree_workspace(int64_t nodes, int32_t heads, int32_t pt_stride) {
  if (tree_shape(nodes, heads, pt_stride)) return -1;
  return paged_workspace(nodes, heads, pt_stride, true);
}

extern "C" int mono_prompt_tree(const mono_prompt_tree_args* args, void* stream) {
  if (!args) return refuse("mono_prompt_tree: args is NULL");
  const mono_prompt_tree_args& a = *args;
  if (int rc = tree_shape(a.nodes, a.heads, a.pt_stride)) return rc;
  if (int rc = need_counts(a.requests, a.pt_stride, a.n_pages)) return rc;
  if (a.nodes == 0) return mono::abi_ok();
  if (int rc = need(a.starts, "starts", 4)) return rc;
  if (a.requests)
    if (int rc = need(a.prefix, "prefix", 4)) return rc;
  if (int rc = need(a.mask, "mask", 8)) return rc;
  Paged p{};
  p.q = a.q, p.tokens = a.nodes, p.heads = a.heads;
  p.starts = a.starts, p.prefix = a.prefix, p.mask = a.mask;
  p.page_table = a.page_table, p.requests = a.requests, p.pt_stride = a.pt_stride, p.n_pages = a.n_pages;
  p.kv = a.kv, p.kv_scale = a.kv_scale, p.out = a.out;
  return run_paged(p, a.pt_stride, a.softmax_scale, a.workspace, a.workspace_bytes, stream);
}
