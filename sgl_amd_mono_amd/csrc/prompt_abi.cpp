// The C entry points of the prompt-width operators: argument checks, the carving of the
// caller's workspace, the launches. They keep no state: every call's scratch is the
// workspace that the call is given.
#include "prompt_abi.h"

namespace {

using namespace mono::prompt;

int need_elements(int64_t rows, int k, const char* names) {
  if (rows * k > MAX_ELEMENTS) return refuse("%s must be at most %lld, got %lld x %d", names, (long long)MAX_ELEMENTS, (long long)rows, k);
  return MONO_OK;
}

int product_shape(int64_t rows, int32_t n, int32_t k) {
  if (int rc = need_rows(rows, "rows")) return rc;
  if (n < 16 || n % 16 || n > MAX_DIM) return refuse("n must be a multiple of 16 in [16, %d], got %d", MAX_DIM, n);
  if (k < BLK || k % BLK || k > MAX_DIM) return refuse("k must be a multiple of %d in [%d, %d], got %d", BLK, BLK, MAX_DIM, k);
  return need_elements(rows, k, "rows x k");
}

// A product's plan over its workspace: the rows' codes and scales, and its parts.
size_t product_space(void* ws, Product& p) {
  Space sp{static_cast<char*>(ws)};
  p.plan = product_plan(p.rows, p.n, p.k, p.f32);
  if (p.plan.kind != ProductPlan::FEW) p.q = sp.rows(p.rows, p.k);
  if (p.plan.splits > 1) p.part = sp.take<float>((size_t)p.plan.splits * p.rows * p.n);
  return sp.off;
}

int experts_shape(const mono_prompt_experts_args& a) {
  if (int rc = need_rows(a.tokens, "tokens")) return rc;
  if (a.experts < 1 || a.experts > MAX_EXPERTS) return refuse("experts must be in [1, %d], got %d", MAX_EXPERTS, a.experts);
  if (a.picks < 1 || a.picks > 64) return refuse("picks must be in [1, 64], got %d", a.picks);
  if (a.tokens * (a.picks + 1) > MAX_ROWS)
    return refuse("tokens x (picks + 1) must be at most %lld, got %lld x %d", (long long)MAX_ROWS, (long long)a.tokens, a.picks + 1);
  if (a.hidden < BLK || a.hidden % BLK || a.hidden > MAX_DIM)
    return refuse("hidden must be a multiple of %d in [%d, %d], got %d", BLK, BLK, MAX_DIM, a.hidden);
  if (a.inter < BLK || a.inter % BLK || a.inter > MAX_DIM / 2)
    return refuse("inter must be a multiple of %d in [%d, %d], got %d", BLK, BLK, MAX_DIM / 2, a.inter);
  return need_elements(a.tokens, a.hidden, "tokens x hidden");
}

// Where the wide tiles take over, by time alone: above FEW_TOKENS tokens with more than
// WIDE_PICKS picks a routed expert on average. Narrow / wide, us a call in a graph:
//
//   hidden x inter, experts, picks   64 tokens   96 tokens   128 tokens  256 tokens  512 tokens
//   7168 x 512, 256, 8               425 / 452   462 / 509   463 / 495   504 / 544   599 / 571
//   7168 x 1024, 64, 8               270 / 290   280 / 296   300 / 298   449 / 310   655 / 351
//   7168 x 2048, 64, 8               523 / 520   541 / 532   574 / 537   827 / 554   1218 / 615
//   7168 x 2048, 16, 4               176 / 180   205 / 192   249 / 194   379 / 213   584 / 281
//   7168 x 512, 32, 8                103 / 101   124 / 127   147 / 132   211 / 139   329 / 179
//   7168 x 512, 8, 4                  64 / 55     67 / 87     74 / 90    111 / 95    175 / 101
//   2048 x 512, 16, 4                 40 / 37     43 / 54     44 / 56     55 / 56     70 / 59
//   1024 x 128, 8, 2                  21 / 27     21 / 38     21 / 40     23 / 40     25 / 42
//
// The two differ in their up products' sums as well: the narrow ones widen the codes to bf16,
// which costs nothing beside the weights' bytes and makes every product exact, the wide ones
// take the FP8 MFMA's 1.4e-5, as the decode launch does. A mid that this carries over a code's
// border moves by a code, so outputs are 0.0017 and 0.0019 to 0.0022 of their norm from 64 bits. A
// caller who wants a token's bits to be its own in any company asks for the narrow tiles (the
// first geometry: 1500 tokens 1036 us for 685, 8192 tokens 4235 for 1595).
constexpr int WIDE_PICKS = 11, FEW_TOKENS = 96;

// The call's plan over its workspace; `e.tiles` bounds the tile list.
size_t experts_plan(const mono_prompt_experts_args& a, void* ws, Experts& e) {
  Space sp{static_cast<char*>(ws)};
  const int64_t picks = a.tokens * a.picks, places = picks + (a.shared ? a.tokens : 0);
  e.wide = !a.batch_invariant && a.tokens > FEW_TOKENS && picks > (int64_t)WIDE_PICKS * a.experts;
  e.bm = e.wide ? 128 : 64;
  e.tiles = (int)all_tiles(a.tokens, picks, a.experts, e.bm, a.shared);
  e.x = sp.rows(a.tokens, a.hidden);
  e.mid_q = sp.rows(places, a.inter);
  e.sorted = Sorted{sp.take<int>(places), sp.take<int>(picks), sp.take<Tile>(e.tiles)};
  e.mid = e.wide ? nullptr : sp.take<float>((size_t)places * a.inter);
  e.part.v = sp.take<uint16_t>((size_t)places * a.hidden);
  e.part.s = sp.take<float>((size_t)places * (a.hidden / PART));
  e.part.ld = a.hidden;
  e.w13 = static_cast<const uint8_t*>(a.w13);
  e.w2 = static_cast<const uint8_t*>(a.w2);
  e.s13 = a.s13;
  e.s2 = a.s2;
  e.weights = a.weights;
  e.residual = a.residual;
  e.residual_stride = a.residual_stride;
  e.out = a.out;
  e.out_stride = a.out_stride;
  e.tokens = a.tokens;
  e.picks = picks;
  e.picks_each = a.picks;
  e.experts = a.experts;
  e.hidden = a.hidden;
  e.inter = a.inter;
  e.shared = a.shared != 0;
  return sp.off;
}

}  // namespace

extern "C" int64_t mono_prompt_product_workspace(int64_t rows, int32_t n, int32_t k) {
  if (product_shape(rows, n, k)) return -1;
  Product p{};
  p.rows = rows, p.n = n, p.k = k;
  mono::abi_ok();
  if (!rows) return 0;
  const size_t bf16 = product_space(nullptr, p);
  p.f32 = true;
  const size_t f32 = product_space(nullptr, p);
  return (int64_t)(bf16 > f32 ? bf16 : f32);
}

extern "C" int mono_prompt_product(const mono_prompt_product_args* args, void* stream) {
  if (!args) return refuse("mono_prompt_product: args is NULL");
  const mono_prompt_product_args& a = *args;
  if (int rc = product_shape(a.rows, a.n, a.k)) return rc;
  if (a.rows == 0) return mono::abi_ok();
  if (int rc = need_stride(a.x_stride, a.k, 8, "x_stride")) return rc;
  if (int rc = need_stride(a.out_stride, a.n, 8, "out_stride")) return rc;
  if (int rc = need(a.x, "x", 16)) return rc;
  if (int rc = need(a.w, "w", 16)) return rc;
  if (int rc = need(a.s, "s", 4)) return rc;
  if (int rc = need(a.out, "out", 16)) return rc;
  Product p{a.x, a.x_stride, {}, a.rows, static_cast<const uint8_t*>(a.w), a.s, a.n, a.k, a.out, a.out_stride, a.out_f32 != 0};
  if (const size_t bytes = product_space(nullptr, p)) {
    if (int rc = need_space(a.workspace, a.workspace_bytes, bytes)) return rc;
    product_space(a.workspace, p);
  }
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (p.plan.kind == ProductPlan::FEW) return launched(few_product(p, st), "the product");
  if (hipError_t e = quant_rows(p.x, false, p.x_stride, p.rows, p.k, p.q, st)) return launched(e, "the rows' rounding");
  if (hipError_t e = p.plan.kind == ProductPlan::WIDE ? wide_product(p, st) : narrow_product(p, st)) return launched(e, "the product");
  return launched(p.plan.splits > 1 ? join_product(p, st) : hipSuccess, "the sum of the product's parts");
}

extern "C" int mono_prompt_append(const mono_prompt_append_args* args, void* stream) {
  return mono_prompt_append_at(args, nullptr, stream);
}

extern "C" int mono_prompt_append_at(const mono_prompt_append_args* args, const int32_t* slot_pos, void* stream) {
  if (!args) return refuse("mono_prompt_append: args is NULL");
  const mono_prompt_append_args& a = *args;
  if (int rc = need_rows(a.tokens, "tokens")) return rc;
  if (a.requests < 0 || a.pt_stride < 0 || a.n_pages < 0 || a.max_pos < 0)
    return refuse("requests, pt_stride, n_pages and max_pos must not be negative, got %d, %d, %d, %d", a.requests, a.pt_stride,
                  a.n_pages, a.max_pos);
  if (a.tokens == 0 || a.requests == 0 || a.pt_stride == 0 || a.n_pages == 0 || a.max_pos == 0) return mono::abi_ok();
  const int each = a.f32 ? 4 : 8;  // a 16-byte load's elements
  if (int rc = need_stride(a.kv_stride, LATENT + PE, each, "kv_stride")) return rc;
  if (int rc = need_stride(a.ik_stride, INDEX, each, "ik_stride")) return rc;
  if (int rc = need(a.kv_a, "kv_a", 16)) return rc;
  if (int rc = need(a.ik, "ik", 16)) return rc;
  if (int rc = need(a.req, "req", 4)) return rc;
  if (int rc = need(a.pos, "pos", 4)) return rc;
  if (int rc = need(a.page_table, "page_table", 4)) return rc;
  if (int rc = need(a.g_kv, "g_kv", 16)) return rc;
  if (int rc = need(a.g_ik, "g_ik", 16)) return rc;
  if (int rc = need(a.b_ik, "b_ik", 16)) return rc;
  if (int rc = need(a.rope_cos, "rope_cos", 16)) return rc;
  if (int rc = need(a.rope_sin, "rope_sin", 16)) return rc;
  if (int rc = need(a.kv, "kv", 8)) return rc;
  if (a.kv_scale)
    if (int rc = need(a.kv_scale, "kv_scale", 4)) return rc;
  if (int rc = need(a.ikv, "ikv", 4)) return rc;
  if (int rc = need(a.iks, "iks", 1)) return rc;
  if (slot_pos)
    if (int rc = need(slot_pos, "slot_pos", 4)) return rc;
  return launched(append(a, slot_pos, static_cast<hipStream_t>(stream)), "the cache append");
}

extern "C" int64_t mono_prompt_experts_workspace(const mono_prompt_experts_args* args) {
  if (!args) return refuse("mono_prompt_experts_workspace: args is NULL"), -1;
  if (experts_shape(*args)) return -1;
  Experts e{};
  mono::abi_ok();
  return (int64_t)experts_plan(*args, nullptr, e);
}

extern "C" int mono_prompt_experts(const mono_prompt_experts_args* args, void* stream) {
  if (!args) return refuse("mono_prompt_experts: args is NULL");
  const mono_prompt_experts_args& a = *args;
  if (int rc = experts_shape(a)) return rc;
  if (a.tokens == 0) return mono::abi_ok();
  if (int rc = need_stride(a.x_stride, a.hidden, 8, "x_stride")) return rc;
  if (int rc = need_stride(a.out_stride, a.hidden, 8, "out_stride")) return rc;
  if (int rc = need(a.x, "x", 16)) return rc;
  if (int rc = need(a.ids, "ids", 4)) return rc;
  if (int rc = need(a.weights, "weights", 4)) return rc;
  if (int rc = need(a.w13, "w13", 16)) return rc;
  if (int rc = need(a.s13, "s13", 4)) return rc;
  if (int rc = need(a.w2, "w2", 16)) return rc;
  if (int rc = need(a.s2, "s2", 4)) return rc;
  if (int rc = need(a.out, "out", 16)) return rc;
  if (a.residual) {
    if (int rc = need_stride(a.residual_stride, a.hidden, 8, "residual_stride")) return rc;
    if (int rc = need(a.residual, "residual", 16)) return rc;
  }
  Experts e{};
  if (int rc = need_space(a.workspace, a.workspace_bytes, experts_plan(a, nullptr, e))) return rc;
  experts_plan(a, a.workspace, e);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (hipError_t r = sort_quant(a.x, a.x_stride, a.tokens, a.hidden, e.x, a.ids, a.picks, a.experts, e.shared, e.bm, e.sorted, st))
    return launched(r, "the tokens' sort");
  if (e.wide) {
    if (hipError_t r = wide_experts_up(e, st)) return launched(r, "the experts' up products");
    if (hipError_t r = wide_experts_down(e, st)) return launched(r, "the experts' down products");
  } else {
    if (hipError_t r = experts_up(e, st)) return launched(r, "the experts' up products");
    if (hipError_t r = experts_down(e, st)) return launched(r, "the experts' down products");
  }
  return launched(experts_back(e, st), "the weighted sum");
}
