// Host-only driver for the sanitizer test: the attention sublayer's planners over
// many random and edge-case requests, under AddressSanitizer and
// UndefinedBehaviorSanitizer, and what has to hold of each plan that is given.
#include <cstdio>
#include <cstring>
#include <random>

#include "../kernels/attention.h"
#include "program.h"

using namespace tiler_rt;

static uint64_t pick(std::mt19937_64& r, uint64_t most) {
  static const uint64_t edges[] = {0, 1, 2, 3, 7, 8, 15, 16, 17, 63, 64, 255, 256, 257, 1023, 1024, 4095, 65536, 1ull << 20,
                                   (1ull << 31) - 2, (1ull << 31) - 1, 1ull << 31, 0xffffffffull, 1ull << 32, 1ull << 40,
                                   UINT64_MAX / 3, UINT64_MAX};
  if (r() % 12 == 0) return edges[r() % (sizeof(edges) / sizeof(edges[0]))];
  uint64_t v = r() % (most + 1);
  return r() % 2 ? v : v >> r() % 12;
}

static bool bad(const char* what) {
  std::printf("%s\n", what);
  return true;
}

static bool check(const Program& p) {
  if (p.nslots > kMaxSlots || p.nlaunches > kMaxLaunches) return bad("too many slots or launches");
  for (uint32_t i = 0; i < p.nlaunches; ++i) {
    const Launch& l = p.launches[i];
    if (l.overflow || l.nargs > kMaxArgs || l.kernarg_bytes > kMaxKernargBytes) return bad("argument segment overflow");
    if (!l.grid[0] || !l.grid[1] || l.grid[1] > 65535 || (uint64_t)l.grid[0] * l.block >= 1ull << 32) return bad("grid");
    for (uint32_t b = 0; b < l.nbindings; ++b)
      if (l.bindings[b].slot >= p.nslots || l.bindings[b].offset + 8 > l.kernarg_bytes) return bad("binding");
  }
  return false;
}

static uint64_t scratch(const Program& p) {
  uint64_t n = 0;
  for (uint32_t i = 0; i < p.nslots; ++i) n += p.slot_roles[i] == kSlotScratch ? p.slot_bytes[i] : 0;
  return n;
}

int main() {
  std::mt19937_64 r(20);
  uint64_t planned = 0, tails = 0, parts = 0;
  for (int it = 0; it < 400000; ++it) {
    static const uint32_t cus[] = {256, 256, 256, 1, 2, 64, 104, 304};
    const Target t{cus[r() % 8], kRowSyncDefaultWaitTicks};
    uintptr_t addr[kMaxSlots] = {};
    if (r() % 8 == 0) addr[r() % 3] = 1 + r() % 16;
    tiler_hip_paged_cache c{};
    c.pages = pick(r, 5000), c.page = (uint32_t)pick(r, 128), c.heads = (uint32_t)pick(r, 16);
    c.head_dim = r() % 8 ? 8 * (1 + r() % 32) : (uint32_t)pick(r, 300);
    const uint64_t row = (uint64_t)c.heads * c.head_dim;
    const bool by_heads = r() % 2;
    c.head_stride = by_heads ? (uint64_t)c.page * c.head_dim : c.head_dim;
    c.token_stride = by_heads ? c.head_dim : row;
    c.page_stride = c.page * row;
    uint64_t* const strides[] = {&c.page_stride, &c.token_stride, &c.head_stride};
    if (r() % 8 == 0) *strides[r() % 3] = pick(r, 1 << 20);
    tiler_hip_attention_shape a{};
    const uint64_t group = r() % 4 ? 1 + r() % 8 : pick(r, 200);
    a.tokens = pick(r, 20000), a.sequences = r() % 4 ? 1 + r() % 64 : pick(r, 2000);
    a.q_heads = (uint32_t)(c.heads * group);
    static const float scales[] = {0.125f, 0.125f, 0.125f, 1e30f, 1e-38f, 0.0f, -1.0f, 3e38f};
    a.scale = scales[r() % 8];
    a.q_stride = (uint64_t)a.q_heads * c.head_dim + (r() % 4 ? 0 : pick(r, 100)), a.out_stride = a.q_stride;
    a.table_width = pick(r, 4000);
    a.window = r() % 2 ? 0 : (uint32_t)pick(r, 40000), a.sinks = r() % 2 ? 0 : (uint32_t)pick(r, 100);
    a.max_fresh = r() % 3 ? pick(r, 3000) : 0, a.max_length = r() % 3 ? pick(r, 200000) : 0;
    static const uint32_t forms[] = {TILER_HIP_FORM_AUTO, TILER_HIP_FORM_AUTO, TILER_HIP_FORM_ATTENTION_FEW,
                                     TILER_HIP_FORM_ATTENTION_TILE_128, TILER_HIP_FORM_ATTENTION_TILE_256};
    Program p;
    if (plan_paged_attention_bf16(t, a, c, addr, p, forms[r() % 5]) == TILER_HIP_OK && p.nlaunches) {
      if (check(p)) return 1;
      TilerAttentionShape s;
      std::memcpy(&s, p.launches[0].kernargs, sizeof(s));
      const Launch& l = p.launches[0];
      const bool few = std::strstr(l.symbol, "few") != nullptr;
      const uint32_t rows = l.block == 512 ? 256 : 128;
      const uint64_t part = 4ull * s.head_dim + 8, all = a.tokens * a.q_heads;
      if (s.splits == 0 || s.whole % s.kv_heads || l.grid[0] < s.whole || (l.grid[0] - s.whole) % s.splits) return bad("parts");
      if ((l.grid[0] - s.whole) / s.splits == 0) return bad("nothing split");
      if (few && (s.whole || l.grid[0] != a.sequences * s.kv_heads * s.splits)) return bad("few rows");
      // every tile that there may be: as many as full rows need, and one for each sequence
      if (!few && s.whole + (l.grid[0] - s.whole) / s.splits != (a.tokens * s.group / rows + a.sequences) * s.kv_heads)
        return bad("tiles");
      if ((s.splits > 1) != (p.nlaunches == 2) || (s.splits == 1 && s.whole)) return bad("join");
      if (scratch(p) != (s.splits == 1 ? 0 : s.whole ? (uint64_t)(l.grid[0] - s.whole) * rows * part : all * s.splits * part))
        return bad("scratch");
      const uint64_t places = (uint64_t)t.compute_units * (rows == 128 && s.head_dim <= 128 ? 2 : 1);
      const uint64_t eight = 8 * all * part, least = eight > 256ull << 20 ? eight : 256ull << 20;
      if (scratch(p) > (s.whole ? 2 * places * rows * part : least)) return bad("scratch past its bound");
      ++planned;
      tails += s.whole != 0;
      parts += s.splits > 1;
    }
    tiler_hip_head_layout h{};
    h.tokens = pick(r, 10000), h.q_heads = (uint32_t)pick(r, 64), h.kv_heads = (uint32_t)pick(r, 16);
    h.head_dim = (uint32_t)pick(r, 1024), h.rotary = r() % 2 ? h.head_dim : (uint32_t)pick(r, 256) & ~1u;
    h.pairing = r() % 3, h.eps_bits = r() % 3 ? 0x358637BDu : (uint32_t)(r() % 2 ? r() : 0);
    h.q_stride = (uint64_t)h.q_heads * h.head_dim + pick(r, 3), h.k_stride = (uint64_t)h.kv_heads * h.head_dim + pick(r, 3);
    h.v_stride = h.k_stride, h.q_out_stride = h.q_stride, h.k_out_stride = h.k_stride;
    if (r() % 2) c.heads = h.kv_heads, c.head_dim = h.head_dim;
    for (uint32_t dtype : {TILER_HIP_F32, TILER_HIP_BF16}) {
      Program f, g, every;
      const uint32_t some = (uint32_t)r() % 128;
      if (plan_norm_rotate(t, dtype, (uint32_t)r() % 8, h, r() % 2 ? &c : nullptr, addr, f) == TILER_HIP_OK && check(f)) return 1;
      planned += f.nlaunches;
      if (plan_norm_rotate_backward(t, dtype, some & ~4u, h, addr, g) != TILER_HIP_OK) continue;
      if (check(g)) return 1;
      // the workspace that the query answers, that of every gradient, holds any of them
      const uint32_t sums = h.eps_bits ? TILER_HIP_ROTATE_DWQ | TILER_HIP_ROTATE_DWK : 0u;
      if (plan_norm_rotate_backward(t, dtype, TILER_HIP_ROTATE_DQ | TILER_HIP_ROTATE_DK | sums, h, addr, every) == TILER_HIP_OK &&
          scratch(g) > scratch(every))
        return bad("workspace of some gradients past that of all");
      planned += g.nlaunches;
    }
    Program q;
    if (plan_page_slots(pick(r, 3000), pick(r, 100000), pick(r, 128), pick(r, 5000), pick(r, 4000), q) == TILER_HIP_OK && check(q))
      return 1;
  }
  if (!tails || !parts) return bad("no parts planned"), 1;
  std::printf("attention-planner-sanitize ok: %llu launches, %llu last rounds in parts\n", (unsigned long long)planned,
              (unsigned long long)tails);
  return 0;
}
