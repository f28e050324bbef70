// Planners of the attention sublayer's families: page tables and cache slots,
// the head norms with the rotation and their gradients, attention over a paged
// cache.
#include "../kernels/attention.h"

#include <algorithm>
#include <cmath>
#include <cstdio>

#include "../kernels/head_rotate.h"
#include "../kernels/page_slots.h"
#include "program.h"

namespace tiler_rt {

namespace {

uint64_t mul_sat(uint64_t a, uint64_t b) { return a && b > UINT64_MAX / a ? UINT64_MAX : a * b; }
uint64_t add_sat(uint64_t a, uint64_t b) { return b > UINT64_MAX - a ? UINT64_MAX : a + b; }
bool aligned16(uintptr_t a) { return (a & 15u) == 0; }
uint64_t ceil_div(uint64_t a, uint64_t b) { return a / b + (a % b != 0); }
constexpr uint64_t kMostPositions = 0x7fffffff;  // positions and slots are int32

const char* type_name(uint32_t dtype) { return dtype == TILER_HIP_BF16 ? "bf16" : "f32"; }

void slot_or_null(Launch& l, bool present, uint32_t slot) {
  if (present) l.ptr(slot);
  else l.null_ptr();
}

// Elements from the first to past the last of `rows` rows of `row` elements.
uint64_t span(uint64_t rows, uint64_t stride, uint64_t row) {
  return rows ? add_sat(mul_sat(rows - 1, stride), row) : 0;
}

TilerDivisor divisor_of(uint32_t d) {
  TilerDivisor v{d, 1, 0};
  while ((1ull << v.shift) < d) ++v.shift;
  v.multiplier = (uint32_t)(((1ull << 32) * ((1ull << v.shift) - d)) / d + 1);
  return v;
}

// A cache's elements from the first to past the last, or a refusal.
tiler_hip_status check_cache(const tiler_hip_paged_cache& c, Program& p, uint64_t& elements) {
  if (c.reserved) return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "paged cache: reserved is not 0");
  if (c.page == 0 || c.heads == 0 || c.head_dim == 0)
    return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "paged cache: empty pages or heads");
  if (mul_sat(c.pages, c.page) > kMostPositions)
    return p.refuse(TILER_HIP_REFUSE_CAPACITY, "paged cache: more than 2^31 - 1 tokens");
  // no two rows overlap: each stride passes what the smaller ones span
  struct Axis {
    uint64_t count, stride;
  } axes[3] = {{c.pages, c.page_stride}, {c.page, c.token_stride}, {c.heads, c.head_stride}};
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2 - i; ++j)
      if (axes[j].count <= 1 ? false : axes[j + 1].count <= 1 || axes[j].stride > axes[j + 1].stride)
        std::swap(axes[j], axes[j + 1]);
  elements = c.head_dim;
  for (const Axis& a : axes) {
    if (a.count <= 1) continue;
    if (a.stride < elements) return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "paged cache: rows overlap");
    elements = add_sat(mul_sat(a.count - 1, a.stride), elements);
  }
  if (elements > (1ull << 60)) return p.refuse(TILER_HIP_REFUSE_CAPACITY, "paged cache: strides beyond 64-bit offsets");
  if (c.pages == 0) elements = 0;
  return TILER_HIP_OK;
}

tiler_hip_status check_heads(uint32_t dtype, uint32_t parts, const tiler_hip_head_layout& h, TilerHeads& k, Program& p) {
  if (dtype != TILER_HIP_F32 && dtype != TILER_HIP_BF16)
    return p.refuse(TILER_HIP_REFUSE_UNSUPPORTED, "norm_rotate dtype");
  if (h.head_dim == 0) return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "heads without elements");
  if (h.head_dim > 1024) return p.refuse(TILER_HIP_REFUSE_CAPACITY, "heads of more than 1024 elements");
  if (h.rotary > h.head_dim || h.rotary % 2)
    return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "rotary: an even number of a head's elements");
  if (h.pairing > TILER_HIP_ROTATE_NEIGHBOURS) return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "rotation pairing");
  if (h.reserved) return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "head layout: reserved is not 0");
  float eps;
  std::memcpy(&eps, &h.eps_bits, 4);
  if (h.eps_bits && (!(eps > 0.0f) || !std::isfinite(eps)))
    return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "eps must be positive and finite, or 0 for no norm");
  if (!h.eps_bits && (parts & (TILER_HIP_ROTATE_WQ | TILER_HIP_ROTATE_WK | TILER_HIP_ROTATE_DWQ | TILER_HIP_ROTATE_DWK)))
    return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "weights without a norm");
  if (h.q_heads > (1u << 20) || h.kv_heads > (1u << 20))
    return p.refuse(TILER_HIP_REFUSE_CAPACITY, "more than 2^20 heads");
  if (h.tokens > (1ull << 40) || h.q_stride > (1ull << 40) || h.k_stride > (1ull << 40) || h.v_stride > (1ull << 40) ||
      h.q_out_stride > (1ull << 40) || h.k_out_stride > (1ull << 40) ||
      mul_sat(h.tokens, h.q_stride + h.k_stride + h.v_stride + h.q_out_stride + h.k_out_stride) > (1ull << 60))
    return p.refuse(TILER_HIP_REFUSE_CAPACITY, "rows of heads beyond 64-bit offsets");
  k = TilerHeads{};
  k.tokens = h.tokens;
  k.q_heads = h.q_heads;
  k.kv_heads = h.kv_heads;
  k.head_dim = h.head_dim;
  k.rotary = h.rotary;
  k.neighbours = h.pairing == TILER_HIP_ROTATE_NEIGHBOURS;
  k.norm = h.eps_bits != 0;
  k.eps = eps;
  k.q_stride = h.q_stride;
  k.k_stride = h.k_stride;
  k.v_stride = h.v_stride;
  k.q_out_stride = h.q_out_stride;
  k.k_out_stride = h.k_out_stride;
  return TILER_HIP_OK;
}

// Lanes that hold a head in units of two 16-byte pieces (head_rotate.hip), or 0 for
// the form of any size: where a piece would be cut, or the head passes a wave.
uint32_t unit_lanes(uint32_t dtype, const tiler_hip_head_layout& h) {
  const uint32_t vec = dtype == TILER_HIP_BF16 ? 8 : 4;
  if (h.head_dim % vec || h.rotary % (2 * vec) || h.rotary / 2 > 512) return 0;
  uint32_t lanes = 4;
  while (lanes * 2 * vec < h.head_dim) lanes *= 2;
  return lanes <= 64 ? lanes : 0;
}

// Tokens a workgroup takes at a time: up to four, whose angles are a good share of
// its threads' first work, once every CU has two workgroups of them.
uint32_t tokens_each(const Target& t, const tiler_hip_head_layout& h) {
  const uint64_t share = h.tokens / (2ull * t.compute_units);
  return share >= 4 ? 4 : share >= 2 ? 2 : 1;
}

}  // namespace

// Slots: [kept, fresh,] [free,] [table,] starts, [lengths,] [positions, slots,]
// taken: those of no elements have none.
tiler_hip_status plan_page_slots(uint64_t sequences, uint64_t tokens, uint64_t page, uint64_t free_count,
                                 uint64_t table_width, Program& p) {
  if (page == 0) return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "page_slots: pages without tokens");
  if (page > kMostPositions || sequences >= kMostPositions || tokens > kMostPositions || free_count > kMostPositions ||
      table_width > kMostPositions)
    return p.refuse(TILER_HIP_REFUSE_CAPACITY, "page_slots: counts of 2^31 and more");
  const bool table = sequences && table_width;
  const uint32_t kept = sequences ? p.slot(4 * sequences, kSlotInput) : 0;
  const uint32_t fresh = sequences ? p.slot(4 * sequences, kSlotInput) : 0;
  const uint32_t free = free_count ? p.slot(4 * free_count, kSlotInput) : 0;
  const uint32_t at = table ? p.slot(4 * sequences * table_width, kSlotOutput) : 0;
  const uint32_t starts = p.slot(4 * (sequences + 1), kSlotOutput);
  const uint32_t lengths = sequences ? p.slot(4 * sequences, kSlotOutput) : 0;
  const uint32_t positions = tokens ? p.slot(4 * tokens, kSlotOutput) : 0;
  const uint32_t slots = tokens ? p.slot(4 * tokens, kSlotOutput) : 0;
  const uint32_t taken = p.slot(4, kSlotOutput);
  TilerPageSlots a{sequences, tokens, free_count, table ? table_width : 0, (uint32_t)page, 0};
  const uint64_t groups = tokens ? ceil_div(tokens, 1024) : 1;
  Launch& l = p.add("tiler_page_slots", (uint32_t)groups, 1, 1024).blob(&a, sizeof(a), 8);
  slot_or_null(l, sequences, kept);
  slot_or_null(l, sequences, fresh);
  slot_or_null(l, free_count, free);
  slot_or_null(l, table, at);
  l.ptr(starts);
  slot_or_null(l, sequences, lengths);
  slot_or_null(l, tokens, positions);
  slot_or_null(l, tokens, slots);
  l.ptr(taken);
  return TILER_HIP_OK;
}

// Slots: [q,] [k,] [v,] [wq,] [wk,] [positions, frequencies,] [q_out,] [k_out,]
// [k_cache, v_cache, slots]: q and k where there are heads, positions and
// frequencies where something is rotated.
tiler_hip_status plan_norm_rotate(const Target& t, uint32_t dtype, uint32_t parts, const tiler_hip_head_layout& h,
                                  const tiler_hip_paged_cache* cache, const uintptr_t*, Program& p) {
  if (parts & ~(uint32_t)(TILER_HIP_ROTATE_WQ | TILER_HIP_ROTATE_WK | TILER_HIP_ROTATE_K_OUT))
    return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "norm_rotate parts");
  TilerHeads a;
  if (tiler_hip_status st = check_heads(dtype, parts, h, a, p); st != TILER_HIP_OK) return st;
  const bool has_q = h.q_heads, has_k = h.kv_heads, k_out = parts & TILER_HIP_ROTATE_K_OUT;
  const uint64_t elem = dtype == TILER_HIP_BF16 ? 2 : 4;
  const uint64_t q_row = (uint64_t)h.q_heads * h.head_dim, k_row = (uint64_t)h.kv_heads * h.head_dim;
  if (h.tokens > 1 && (h.q_stride < q_row || h.k_stride < k_row || h.q_out_stride < q_row ||
                       (k_out && h.k_out_stride < k_row) || (cache && h.v_stride < k_row)))
    return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "rows of heads overlap");
  if (has_k && !k_out && !cache) return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "the keys go nowhere");
  uint64_t cached = 0;
  if (cache) {
    if (dtype != TILER_HIP_BF16) return p.refuse(TILER_HIP_REFUSE_UNSUPPORTED, "the paged cache is bf16");
    if (tiler_hip_status st = check_cache(*cache, p, cached); st != TILER_HIP_OK) return st;
    if (cache->heads != h.kv_heads || cache->head_dim != h.head_dim)
      return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "the cache has other heads");
    a.page = cache->page;
    a.slots = cache->pages * cache->page;
    a.page_stride = cache->page_stride;
    a.token_stride = cache->token_stride;
    a.head_stride = cache->head_stride;
  }
  auto given = [&](bool there, uint64_t bytes, uint32_t role) { return there ? p.slot(bytes, role) : 0; };
  const bool wq = parts & TILER_HIP_ROTATE_WQ, wk = parts & TILER_HIP_ROTATE_WK;
  const uint32_t q = given(has_q, mul_sat(span(h.tokens, h.q_stride, q_row), elem), kSlotInput);
  const uint32_t k = given(has_k, mul_sat(span(h.tokens, h.k_stride, k_row), elem), kSlotInput);
  const uint32_t v = given(cache, mul_sat(span(h.tokens, h.v_stride, k_row), elem), kSlotInput);
  const uint32_t at_wq = given(wq, elem * h.head_dim, kSlotInput), at_wk = given(wk, elem * h.head_dim, kSlotInput);
  const uint32_t positions = given(h.rotary, mul_sat(h.tokens, 4), kSlotInput);
  const uint32_t frequencies = given(h.rotary, 4ull * h.rotary, kSlotInput);
  const uint32_t q_out = given(has_q, mul_sat(span(h.tokens, h.q_out_stride, q_row), elem), kSlotOutput);
  const uint32_t to_k = given(k_out, mul_sat(span(h.tokens, h.k_out_stride, k_row), elem), kSlotOutput);
  const uint32_t k_cache = given(cache, cached * 2, kSlotOutput), v_cache = given(cache, cached * 2, kSlotOutput);
  const uint32_t slots = given(cache, mul_sat(h.tokens, 4), kSlotInput);
  if (h.tokens == 0 || (!has_q && !has_k)) return TILER_HIP_OK;
  char name[64];
  const uint32_t lanes = unit_lanes(dtype, h);
  a.each = lanes ? tokens_each(t, h) : 1;
  const uint64_t all = ceil_div(h.tokens, a.each);
  const uint32_t groups = (uint32_t)(all < (1u << 20) ? all : 1u << 20);
  if (lanes) std::snprintf(name, sizeof(name), "tiler_norm_rotate_%s_%c%u", type_name(dtype), a.neighbours ? 'n' : 'h', lanes);
  else std::snprintf(name, sizeof(name), "tiler_norm_rotate_%s_any", type_name(dtype));
  // few tokens: workgroups that share one's heads, one a group of lanes, up to two a CU
  uint64_t share = 1;
  if (lanes && groups < 2 * t.compute_units) {
    const uint64_t heads = (uint64_t)h.q_heads + h.kv_heads + (cache ? h.kv_heads : 0);
    share = ceil_div(a.each * heads * lanes, 256);
    if (share > 2 * t.compute_units / groups) share = 2 * t.compute_units / groups;
  }
  Launch& l = p.add(name, groups, (uint32_t)share, 256).blob(&a, sizeof(a), 8);
  slot_or_null(l, has_q, q);
  slot_or_null(l, has_k, k);
  slot_or_null(l, cache, v);
  slot_or_null(l, wq, at_wq);
  slot_or_null(l, wk, at_wk);
  slot_or_null(l, h.rotary, positions);
  slot_or_null(l, h.rotary, frequencies);
  slot_or_null(l, has_q, q_out);
  slot_or_null(l, k_out, to_k);
  slot_or_null(l, cache, k_cache);
  slot_or_null(l, cache, v_cache);
  slot_or_null(l, cache, slots);
  return TILER_HIP_OK;
}

// Slots: [dq_out,] [dk_out,] [q, k,] [wq,] [wk,] [positions, frequencies,] [dq,]
// [dk,] [dwq,] [dwk,] [partials: scratch]: q and k where there is a norm.
tiler_hip_status plan_norm_rotate_backward(const Target& t, uint32_t dtype, uint32_t parts,
                                           const tiler_hip_head_layout& h, const uintptr_t*, Program& p) {
  const uint32_t known = TILER_HIP_ROTATE_WQ | TILER_HIP_ROTATE_WK | TILER_HIP_ROTATE_DQ | TILER_HIP_ROTATE_DK |
                         TILER_HIP_ROTATE_DWQ | TILER_HIP_ROTATE_DWK;
  if (parts & ~known) return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "norm_rotate_backward parts");
  TilerHeads a;
  if (tiler_hip_status st = check_heads(dtype, parts, h, a, p); st != TILER_HIP_OK) return st;
  const bool wq = parts & TILER_HIP_ROTATE_WQ, wk = parts & TILER_HIP_ROTATE_WK;
  const bool dwq = parts & TILER_HIP_ROTATE_DWQ, dwk = parts & TILER_HIP_ROTATE_DWK;
  const bool dq = (parts & TILER_HIP_ROTATE_DQ) && h.q_heads, dk = (parts & TILER_HIP_ROTATE_DK) && h.kv_heads;
  const bool of_q = (dq || dwq) && h.q_heads, of_k = (dk || dwk) && h.kv_heads;
  const uint64_t elem = dtype == TILER_HIP_BF16 ? 2 : 4;
  const uint64_t q_row = (uint64_t)h.q_heads * h.head_dim, k_row = (uint64_t)h.kv_heads * h.head_dim;
  if (h.tokens > 1 && ((of_q && (h.q_stride < q_row || h.q_out_stride < q_row)) ||
                       (of_k && (h.k_stride < k_row || h.k_out_stride < k_row))))
    return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "rows of heads overlap");
  auto given = [&](bool there, uint64_t bytes, uint32_t role) { return there ? p.slot(bytes, role) : 0; };
  const uint32_t dq_out = given(of_q, mul_sat(span(h.tokens, h.q_out_stride, q_row), elem), kSlotInput);
  const uint32_t dk_out = given(of_k, mul_sat(span(h.tokens, h.k_out_stride, k_row), elem), kSlotInput);
  const uint32_t q = given(of_q && a.norm, mul_sat(span(h.tokens, h.q_stride, q_row), elem), kSlotInput);
  const uint32_t k = given(of_k && a.norm, mul_sat(span(h.tokens, h.k_stride, k_row), elem), kSlotInput);
  const uint32_t at_wq = given(wq, elem * h.head_dim, kSlotInput), at_wk = given(wk, elem * h.head_dim, kSlotInput);
  const uint32_t positions = given(h.rotary, mul_sat(h.tokens, 4), kSlotInput);
  const uint32_t frequencies = given(h.rotary, 4ull * h.rotary, kSlotInput);
  const uint32_t at_dq = given(dq, mul_sat(span(h.tokens, h.q_stride, q_row), elem), kSlotOutput);
  const uint32_t at_dk = given(dk, mul_sat(span(h.tokens, h.k_stride, k_row), elem), kSlotOutput);
  const uint32_t at_dwq = given(dwq, elem * h.head_dim, kSlotOutput), at_dwk = given(dwk, elem * h.head_dim, kSlotOutput);
  char name[64];
  const bool sum_q = of_q && dwq && h.tokens, sum_k = of_k && dwk && h.tokens;
  uint32_t partials_q = 0, partials_k = 0;
  // Each workgroup leaves one row of partial sums.  In units, four to a CU, by the
  // heads' shares; the form of any size, whose four waves take a head each, as many
  // as LDS holds, by the rounds of heads: a token's way through it is latency (1237
  // tokens of 7 and 1 heads of 90 f32, us traced: 9.1, at half as many, one half of them
  // the keys', 14.4).
  const uint32_t lanes = unit_lanes(dtype, h);
  a.each = lanes ? tokens_each(t, h) : 1;
  const uint64_t most = (lanes ? 4ull : 8ull) * t.compute_units, all = ceil_div(h.tokens, a.each);
  const double of_each_q = lanes ? h.q_heads : (double)ceil_div(h.q_heads, 4);
  const double of_each_k = lanes ? h.kv_heads : (double)ceil_div(h.kv_heads, 4);
  const double share = of_q && of_k ? of_each_q / (of_each_q + of_each_k) : 1.0;
  const uint64_t q_most = (uint64_t)(share * (double)most), k_most = of_q ? most - q_most : most;
  const uint32_t count_q = of_q ? (uint32_t)(all < q_most ? all : q_most ? q_most : 1) : 0;
  const uint32_t count_k = of_k ? (uint32_t)(all < k_most ? all : k_most ? k_most : 1) : 0;
  a.q_groups = count_q;
  if (sum_q) partials_q = p.slot(4ull * count_q * h.head_dim, kSlotScratch);
  if (sum_k) partials_k = p.slot(4ull * count_k * h.head_dim, kSlotScratch);
  if (h.tokens && (of_q || of_k)) {
    if (lanes) std::snprintf(name, sizeof(name), "tiler_norm_rotate_grad_%s_%c%u", type_name(dtype), a.neighbours ? 'n' : 'h', lanes);
    else std::snprintf(name, sizeof(name), "tiler_norm_rotate_grad_%s_any", type_name(dtype));
    Launch& l = p.add(name, count_q + count_k, 1, 256).blob(&a, sizeof(a), 8);
    slot_or_null(l, of_q, dq_out);
    slot_or_null(l, of_k, dk_out);
    slot_or_null(l, of_q && a.norm, q);
    slot_or_null(l, of_k && a.norm, k);
    slot_or_null(l, wq, at_wq);
    slot_or_null(l, wk, at_wk);
    slot_or_null(l, h.rotary, positions);
    slot_or_null(l, h.rotary, frequencies);
    slot_or_null(l, dq, at_dq);
    slot_or_null(l, dk, at_dk);
    slot_or_null(l, sum_q, partials_q);
    slot_or_null(l, sum_k, partials_k);
  }
  if (dwq || dwk) {  // no tokens or no heads: zeros
    std::snprintf(name, sizeof(name), "tiler_norm_rotate_sum_%s", type_name(dtype));
    Launch& l = p.add(name, (uint32_t)ceil_div(h.head_dim, 16), 2, 1024);
    slot_or_null(l, sum_q, partials_q);
    slot_or_null(l, sum_k, partials_k);
    l.u32(sum_q ? count_q : 0).u32(sum_k ? count_k : 0).u32(h.head_dim);
    slot_or_null(l, dwq, at_dwq);
    slot_or_null(l, dwk, at_dwk);
  }
  return TILER_HIP_OK;
}

namespace {

// A form of the attention's tiles: rows, the head size it is built for, the tiles of
// a batch (at most: each sequence's last one may be cut) and the parts of the keys.
struct AttentionForm {
  uint32_t rows, dim;
  uint64_t tiles, splits;
  uint64_t whole;  // of the tiles times heads: those that are not split (0: all are)
};

// us a step of 64 keys takes where a CU has one workgroup, and where it has two
// (128 rows; LDS holds one from heads of more than 128 on), or eight waves of 256 rows:
// 512, 4096 and 8192 rows a head over 8000 keys and more, pages of 64.
struct StepTime {
  uint32_t dim;
  double one, two, eight_alone, eight;
};
constexpr StepTime kStepTimes[] = {
    {64, 0.93, 1.30, 1.10, 1.25}, {96, 1.10, 1.66, 1.33, 1.45}, {128, 1.25, 2.00, 1.55, 1.80},
    {192, 2.05, 0, 0, 0},         {256, 2.70, 0, 0, 0},
};

AttentionForm choose_attention(const Target& t, uint64_t tokens, uint64_t sequences, uint64_t fresh, uint32_t heads,
                               uint32_t group, uint32_t head_dim, uint64_t longest, uint64_t window, uint32_t form) {
  const uint64_t cus = t.compute_units, rows = tokens * group;
  // Parts of all rows, results in binary32: eight (16 times the output) at most, or
  // 256 MB of them, which eight rounds of full tiles leave (256 CUs).
  const uint64_t most_parts = std::max<uint64_t>(8, (256ull << 20) / (rows * heads * (head_dim * 4 + 8)));
  if (form == TILER_HIP_FORM_AUTO ? fresh * group <= 16 : form == TILER_HIP_FORM_ATTENTION_FEW) {
    // One turn of 16 rows (32 rows, two turns, us: 90, in tiles of 128 rows 58; 16 rows 25.2
    // and 24.8; 2 rows 14.5 and 14.8; 4 rows over 32000 keys 164 and 167).  Two workgroups
    // to a CU, 256 keys at least to a part: 16 sequences of up to 1000 keys, 8 heads, whole /
    // in two / four / eight parts 19.1 / 16.0 / 14.5 / 16.2; 8 of up to 32000, in two / four /
    // eight / sixteen 232 / 160 / 164 / 164.
    const uint64_t seen = window && longest > window ? window : longest;
    uint64_t splits = ceil_div(2 * cus, mul_sat(sequences, heads));
    if (splits > ceil_div(seen, 256)) splits = ceil_div(seen, 256);
    // A part's time falls with their number and the join's grows with it, us for one
    // sequence on one key/value head of 128 in half / as many / twice / four times as
    // many parts: 8000 keys (31) 18.5 / 17.0 / 18.4 / 24.6, 32000 (63) 29.3 / 24.7 / 29.0 /
    // 42.9, 130000 (127) 49.7 / 42.3 / 53.4 / 84; 32000 and 130000 on two heads 30.6 / 25.6
    // / 31.6 and 52.3 / 49.8 / 63.7, on eight (the CUs' share) 38.0 / 40.3 and 105 / 110.
    const uint64_t most = (uint64_t)std::sqrt((double)seen / 8.0);
    if (splits > most) splits = most;
    if (splits > most_parts) splits = most_parts;
    return {16, head_dim <= 64 ? 64u : head_dim <= 128 ? 128u : 256u, sequences, splits ? splits : 1, 0};
  }
  // The least of an estimate: a part's steps, and two for its start and end, in the
  // rounds that its workgroups take; past the first round the average length counts,
  // and a tail, of the longest less what a prompt's rows, the last ones first, level out.
  // A lone sequence's average is its middle row's; that of several, of which nothing but
  // the longest is known, half of that.  Parts cost a launch and their results' way out
  // and back.  The constants are the least regret (under 1 % on average) over 18
  // batches measured in both tiles and 1 to 16 parts.
  // us, 512 tokens of 32 and 8 heads of 128 over 8512 keys: 128 rows whole 169, in two /
  // three / four / six parts 96 / 93 / 85 / 94; 256 rows in four 81.  Two prompts of 4096:
  // 256 rows 282, 128 rows 293.  24 sequences of up to 150 tokens over up to 3000 keys, 35
  // and 5 heads of 80: 128 rows whole, in two / three / four / six 69 / 62 / 60 / 61 / 75.
  const StepTime* c = kStepTimes;
  while (c->dim < head_dim) ++c;
  AttentionForm best{};
  double least = 0;
  for (const uint32_t tile : {128u, 256u}) {
    if (tile == 256 && head_dim > 128) continue;
    if (form != TILER_HIP_FORM_AUTO && (tile == 256) != (form == TILER_HIP_FORM_ATTENTION_TILE_256)) continue;
    const double one = tile == 256 ? c->eight_alone : c->one, two = tile == 256 ? c->eight : c->two > 0 ? c->two : c->one;
    const double slots = (double)cus * (tile == 128 && c->two > 0 ? 2 : 1);
    const double each = (double)sequences * (double)ceil_div(fresh * group, tile);
    double tiles = (double)ceil_div(rows, tile) + 0.3 * (double)(sequences - 1);
    if (tokens == sequences * fresh || tiles > each) tiles = each;
    // no two sequences share a tile
    const double own = (double)(sequences < tokens ? sequences : tokens), equal = (tiles > own ? tiles : own) * heads;
    double most = (double)longest, average = most - 0.5 * (double)(fresh < longest ? fresh : longest);
    if (sequences > 1 && average > 0.5 * most) average = 0.5 * most;
    const double shared = window && most > (double)window ? (double)window : most;  // by the parts
    if (const double seen = (double)window + tile / (double)group; window && most > seen) {
      most = seen;
      average = average < seen ? average : seen;
    }
    const double leveled = (double)fresh < most ? (double)fresh : most;
    for (uint64_t splits = 1; splits <= 64 && splits <= most_parts && (splits == 1 || shared >= 256.0 * (double)splits); splits += 1 + splits / 8) {
      const double groups = tiles * heads * (double)splits, by = 64.0 * (double)splits;
      const double beside_us = 0.8 * (most / by + 2) * two;
      double us = (most / by + 2) * one;
      if (groups > slots) us = groups / slots * (average / by + 2) * two + 0.5 * ((most - 0.6 * leveled) / by + 2) * one;
      else if (groups > (double)cus && beside_us > us) us = beside_us;
      if (splits > 1) us += 4 + (double)rows * heads * (double)splits * head_dim * 2e-6;
      if (splits == 1 && equal > slots && average > 0.9 * most) continue;  // below
      if (!best.rows || us < least) best = {tile, c->dim, rows / tile + sequences, splits, 0}, least = us;
    }
    // Equal tiles of more than one round take whole rounds; a last one that fills the CUs
    // badly is split over them.  What is split is every tile that there may be behind the
    // whole ones, most of them empty where sequences are many: their parts, and with them
    // the scratch, are held to two rounds (67 MB on 256 CUs).
    if (equal > slots && average > 0.9 * most) {
      const double rounds = std::floor(equal / slots), rest = equal - rounds * slots;
      const double first_us = rounds * (most / 64 + 2) * two;
      double us = first_us;
      if (rest > 0) us += rest <= (double)cus ? (most / 64 + 2) * one : 0.8 * (most / 64 + 2) * two;
      if (!best.rows || us < least) best = {tile, c->dim, rows / tile + sequences, 1, 0}, least = us;
      const uint64_t whole = (uint64_t)(rounds * slots) / heads * heads, all = (rows / tile + sequences) * heads;
      double parts = rest > 0 ? std::floor(slots / std::ceil(rest)) : 1;
      if (parts > std::floor(shared / 256)) parts = std::floor(shared / 256);
      const double places = whole < all ? std::floor(2 * slots / (double)(all - whole)) : 1;
      if (parts > places) parts = places;
      if (parts < 2 || !whole) continue;
      us = first_us + (most / 64 / parts + 2) * (rest * parts > (double)cus ? 0.8 * two : one) + 4 +
           rest * tile * parts * head_dim * 2e-6;
      if (us < least) best = {tile, c->dim, rows / tile + sequences, (uint64_t)parts, whole}, least = us;
    }
  }
  return best;
}

}  // namespace

// Slots: q, k, v, [table,] starts, lengths, out, [partial results, their maxima
// and sums: scratch].
tiler_hip_status plan_paged_attention_bf16(const Target& t, const tiler_hip_attention_shape& a,
                                           const tiler_hip_paged_cache& cache, const uintptr_t* addr, Program& p,
                                           uint32_t form) {
  uint64_t cached = 0;
  if (tiler_hip_status st = check_cache(cache, p, cached); st != TILER_HIP_OK) return st;
  if (a.reserved) return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "attention shape: reserved is not 0");
  if (a.q_heads == 0 || a.q_heads % cache.heads)
    return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "query heads: a multiple of the cache's heads");
  if (cache.head_dim % 8 || cache.head_dim > 256)
    return p.refuse(TILER_HIP_REFUSE_UNSUPPORTED, "heads of 8 to 256 elements, a multiple of 8");
  const float scale = (float)((double)a.scale * 1.4426950408889634074);  // of powers of two
  if (!(a.scale > 0.0f) || !std::isfinite(scale))
    return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "scale must be positive and finite");
  if (form != TILER_HIP_FORM_AUTO && (form < TILER_HIP_FORM_ATTENTION_FEW || form > TILER_HIP_FORM_ATTENTION_TILE_256))
    return p.refuse(TILER_HIP_REFUSE_UNSUPPORTED, "form: not one of attention's");
  if (form == TILER_HIP_FORM_ATTENTION_TILE_256 && cache.head_dim > 128)
    return p.refuse(TILER_HIP_REFUSE_UNSUPPORTED, "head-size: tiles of 256 rows hold heads of up to 128 elements");
  const uint64_t row = (uint64_t)a.q_heads * cache.head_dim;
  if (a.tokens > 1 && (a.q_stride < row || a.out_stride < row))
    return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "rows of heads overlap");
  if (a.sequences >= kMostPositions || mul_sat(a.tokens, a.q_heads) > kMostPositions ||
      mul_sat(a.table_width, cache.page) > kMostPositions || a.q_stride > (1ull << 32) || a.out_stride > (1ull << 32))
    return p.refuse(TILER_HIP_REFUSE_CAPACITY, "paged attention: counts of 2^31 and more");
  const bool table = a.sequences && a.table_width;
  const uint32_t q = p.slot(2 * span(a.tokens, a.q_stride, row), kSlotInput);
  const uint32_t k = p.slot(2 * cached, kSlotInput), v = p.slot(2 * cached, kSlotInput);
  const uint32_t at = table ? p.slot(4 * a.sequences * a.table_width, kSlotInput) : 0;
  const uint32_t starts = p.slot(4 * (a.sequences + 1), kSlotInput), lengths = p.slot(4 * a.sequences, kSlotInput);
  const uint32_t out = p.slot(2 * span(a.tokens, a.out_stride, row), kSlotOutput);
  if (a.sequences == 0 || a.tokens == 0) return TILER_HIP_OK;
  // an axis of one has no stride; a page's tokens are stepped through by it all the same
  const uint64_t page_stride = cache.pages > 1 ? cache.page_stride : 0, head_stride = cache.heads > 1 ? cache.head_stride : 0;
  const uint64_t token_stride = cache.page > 1 ? cache.token_stride : 8;
  // the kernels' offsets inside the cache: 32 bits times 32 bits, and 32 inside a page
  if (page_stride > 0xffffffffull || mul_sat(cache.page, token_stride) > 0xffffffffull)
    return p.refuse(TILER_HIP_REFUSE_CAPACITY, "paged attention: a page of 2^32 elements and more");
  if ((page_stride | token_stride | head_stride) % 8 || !aligned16(addr[k]) || !aligned16(addr[v]))
    return p.refuse(TILER_HIP_REFUSE_UNSUPPORTED, "the cache's rows start on 16 bytes");
  TilerAttentionShape s{};
  s.tokens = (uint32_t)a.tokens;
  s.sequences = (uint32_t)a.sequences;
  s.kv_heads = cache.heads;
  s.group = a.q_heads / cache.heads;
  s.head_dim = cache.head_dim;
  s.pages = (uint32_t)cache.pages;
  s.width = (uint32_t)a.table_width;
  s.window = a.window;
  s.sinks = a.sinks;
  s.scale = scale;
  s.page = divisor_of(cache.page);
  s.groups = divisor_of(s.group);
  s.q_stride = a.q_stride;
  s.out_stride = a.out_stride;
  s.page_stride = (uint32_t)page_stride;
  s.token_stride = (uint32_t)token_stride;
  s.head_stride = head_stride;
  const uint64_t room = a.table_width * cache.page;
  uint64_t longest = a.max_length && a.max_length < room ? a.max_length : room;
  const uint64_t window = a.window ? (uint64_t)a.window + a.sinks : 0;
  const uint64_t fresh = a.max_fresh && a.max_fresh < a.tokens ? a.max_fresh : a.tokens;
  const AttentionForm f = choose_attention(t, a.tokens, a.sequences, fresh, cache.heads, s.group, s.head_dim, longest, window, form);
  const uint64_t splits = f.splits, alone = mul_sat(f.tiles, s.kv_heads);
  const uint64_t whole = f.whole < alone ? f.whole : 0, split = alone - whole;  // tiles times heads
  s.splits = (uint32_t)splits;
  s.whole = (uint32_t)whole;
  if (mul_sat(alone, splits) > 0xffffffffull / 512)
    return p.refuse(TILER_HIP_REFUSE_CAPACITY, "paged attention: more workgroups than a launch holds");
  const uint64_t rows = a.tokens * a.q_heads, part_rows = (whole ? split * f.rows : rows) * splits;
  const uint32_t part = splits > 1 ? p.slot(4 * mul_sat(part_rows, s.head_dim), kSlotScratch) : 0;
  const uint32_t ml = splits > 1 ? p.slot(8 * part_rows, kSlotScratch) : 0;
  char name[64];
  if (f.rows == 16) std::snprintf(name, sizeof(name), "tiler_paged_attention_bf16_few%u", f.dim);
  else std::snprintf(name, sizeof(name), "tiler_paged_attention_bf16_t%u_d%u", f.rows, f.dim);
  Launch& l = p.add(name, (uint32_t)(whole + split * splits), 1, f.rows == 256 ? 512 : 256).blob(&s, sizeof(s), 8).ptr(q).ptr(k).ptr(v);
  slot_or_null(l, table, at);
  l.ptr(starts).ptr(lengths).ptr(out);
  slot_or_null(l, splits > 1, part);
  slot_or_null(l, splits > 1, ml);
  if (splits > 1 && whole) {
    std::snprintf(name, sizeof(name), "tiler_paged_attention_bf16_join_t%u", f.rows);
    p.add(name, (uint32_t)split, f.rows / 32, 256).blob(&s, sizeof(s), 8).ptr(starts).ptr(lengths).ptr(part).ptr(ml).ptr(out);
  } else if (splits > 1) {
    const uint64_t groups = ceil_div(rows * (s.head_dim / 4), 256);
    p.add("tiler_paged_attention_bf16_join", (uint32_t)(groups < 16384 ? groups : 16384), 1, 256)
        .blob(&s, sizeof(s), 8).ptr(starts).ptr(part).ptr(ml).ptr(out);
  }
  return TILER_HIP_OK;
}

}  // namespace tiler_rt
