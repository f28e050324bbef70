// Planners of the feed-forward sublayer's families: layer norm and its
// gradients, the gated product and its gradients, the 8-bit linear layer.
#include "program.h"

#include <cmath>
#include <cstdio>

namespace tiler_rt {

namespace {

uint64_t mul_sat(uint64_t a, uint64_t b) { return a && b > UINT64_MAX / a ? UINT64_MAX : a * b; }
bool aligned16(uintptr_t a) { return (a & 15u) == 0; }
uint64_t ceil_div(uint64_t a, uint64_t b) { return a / b + (a % b != 0); }

// Whether one launch holds this many workgroups along x: the runtime takes
// fewer than 2^32 work items.
bool grid_holds(uint64_t workgroups, uint32_t threads) { return workgroups <= 0xffffffffull / threads; }

const char* type_name(uint32_t dtype) { return dtype == TILER_HIP_BF16 ? "bf16" : "f32"; }

void slot_or_null(Launch& l, bool present, uint32_t slot) {
  if (present) l.ptr(slot);
  else l.null_ptr();
}

constexpr uint32_t kRowWorkgroups = 1u << 20;  // rows beyond take further rounds of the streamed forms' row loops
constexpr uint32_t kColumnWorkgroups = 1u << 20;  // and groups of columns of the column sums' loops
uint32_t column_groups(uint64_t extent, uint64_t columns) {
  const uint64_t groups = ceil_div(extent, columns);
  return (uint32_t)(groups < kColumnWorkgroups ? groups : kColumnWorkgroups);
}

// The register form of a row kernel (row_pieces.h) for rows of `extent`
// elements, kVec = `vec` to a 16-byte piece: WAVES waves per row and CH pieces
// a thread, "w{WAVES}c{CH}", or "s" (streamed) beyond what registers hold and for
// rows shorter than a piece.  One wave a row (four rows a workgroup, no barrier)
// where a thread has at most `one_wave` pieces and the rows fill the CUs twice over
// for each; else four waves a row, and sixteen beyond 1024 pieces or for up to a
// row a CU.  us, norm bf16, one wave / four / sixteen: 4096 x 2048 (4 pieces) 8.7 /
// 10.9 / 27, 1024 x 2048 6.5 / 5.4 / 9.3, 8192 x 4096 (8) 31 / 28 / 56; four /
// sixteen: 128 x 8192 6.1 / 4.9, 1024 x 8192 9.6 / 11.4; quantization of bf16 rows,
// 4096 x 2048 (4) 9.5 / 8.4.
struct RowForm {
  char name[16];
  uint32_t block;
  uint64_t grid;
};
RowForm row_form(const Target& t, uint64_t rows, uint64_t extent, uint64_t vec, uint64_t one_wave) {
  const uint64_t pieces = ceil_div(extent, vec);
  RowForm f{"s", 256, rows < kRowWorkgroups ? rows : kRowWorkgroups};
  uint32_t waves = 0, ch = 0;
  auto pow2 = [](uint64_t v) {
    uint32_t p = 1;
    while (p < v) p <<= 1;
    return p;
  };
  const uint32_t alone = pow2(ceil_div(pieces, 64));  // pieces a thread of a row's only wave
  if (extent < vec) waves = 0;
  else if (alone == 1 || (alone <= one_wave && rows >= 2ull * alone * t.compute_units)) waves = 1, ch = alone;
  else if (pieces <= 512 || (pieces <= 1024 && rows > t.compute_units)) waves = 4, ch = pow2(ceil_div(pieces, 256));
  else if (pieces <= 1024 * 4) waves = 16, ch = pow2(ceil_div(pieces, 1024));
  const uint32_t block = waves == 1 ? 256 : 64 * waves;
  const uint64_t grid = waves == 1 ? ceil_div(rows, 4) : rows;
  if (waves && grid_holds(grid, block)) {
    std::snprintf(f.name, sizeof(f.name), "w%uc%u", waves, ch);
    f.block = block;
    f.grid = grid;
  }
  return f;
}

}  // namespace

// Slots: x, [w,] [b,] y, [mean, rstd].
tiler_hip_status plan_layer_norm(const Target& t, uint32_t dtype, uint32_t parts, uint64_t rows, uint64_t extent,
                                 uint32_t eps_bits, const uintptr_t*, Program& p) {
  float eps;
  std::memcpy(&eps, &eps_bits, 4);
  if (!(eps > 0.0f) || !std::isfinite(eps))
    return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "eps must be positive and finite");
  if (dtype != TILER_HIP_F32 && dtype != TILER_HIP_BF16)
    return p.refuse(TILER_HIP_REFUSE_UNSUPPORTED, "layer_norm dtype");
  if (parts & ~(uint32_t)(TILER_HIP_NORM_WEIGHT | TILER_HIP_NORM_BIAS | TILER_HIP_NORM_STATISTICS))
    return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "layer_norm parts");
  const bool has_w = parts & TILER_HIP_NORM_WEIGHT, has_b = parts & TILER_HIP_NORM_BIAS,
             stats = parts & TILER_HIP_NORM_STATISTICS;
  const uint64_t elem = dtype == TILER_HIP_BF16 ? 2 : 4, bytes = mul_sat(mul_sat(rows, extent), elem);
  const uint32_t x = p.slot(bytes, kSlotInput);
  const uint32_t w = has_w ? p.slot(mul_sat(extent, elem), kSlotInput) : 0;
  const uint32_t b = has_b ? p.slot(mul_sat(extent, elem), kSlotInput) : 0;
  const uint32_t y = p.slot(bytes, kSlotOutput);
  const uint32_t mean = stats ? p.slot(mul_sat(rows, 4), kSlotOutput) : 0;
  const uint32_t rstd = stats ? p.slot(mul_sat(rows, 4), kSlotOutput) : 0;
  if (rows && extent == 0 && stats)
    return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "rows without elements have no mean");
  if (rows == 0 || extent == 0) return TILER_HIP_OK;
  if (extent > 0xffffffffull) return p.refuse(TILER_HIP_REFUSE_CAPACITY, "row longer than 2^32 - 1 elements");
  char name[64];
  const RowForm f = row_form(t, rows, extent, 16 / elem, 4);
  std::snprintf(name, sizeof(name), "tiler_layer_norm_%s_%s", type_name(dtype), f.name);
  Launch& l = p.add(name, (uint32_t)f.grid, 1, f.block).ptr(x);
  slot_or_null(l, has_w, w);
  slot_or_null(l, has_b, b);
  l.u64(rows).u64(extent).f32(eps).ptr(y);
  slot_or_null(l, stats, mean);
  slot_or_null(l, stats, rstd);
  return TILER_HIP_OK;
}

// Slots: dy, x, [w,] mean, rstd, [dx,] [dw,] [db,] [partials: scratch].
tiler_hip_status plan_layer_norm_backward(const Target& t, uint32_t dtype, uint32_t parts, uint64_t rows,
                                          uint64_t extent, const uintptr_t*, Program& p) {
  if (dtype != TILER_HIP_F32 && dtype != TILER_HIP_BF16)
    return p.refuse(TILER_HIP_REFUSE_UNSUPPORTED, "layer_norm dtype");
  const uint32_t known = TILER_HIP_NORM_WEIGHT | TILER_HIP_NORM_DX | TILER_HIP_NORM_DW | TILER_HIP_NORM_DB;
  if (parts & ~known) return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "layer_norm_backward parts");
  const bool has_w = parts & TILER_HIP_NORM_WEIGHT, has_dx = parts & TILER_HIP_NORM_DX,
             has_dw = parts & TILER_HIP_NORM_DW, has_db = parts & TILER_HIP_NORM_DB;
  const uint64_t elem = dtype == TILER_HIP_BF16 ? 2 : 4, bytes = mul_sat(mul_sat(rows, extent), elem);
  const uint32_t dy = p.slot(bytes, kSlotInput), x = p.slot(bytes, kSlotInput);
  const uint32_t w = has_w ? p.slot(mul_sat(extent, elem), kSlotInput) : 0;
  const uint32_t mean = p.slot(mul_sat(rows, 4), kSlotInput), rstd = p.slot(mul_sat(rows, 4), kSlotInput);
  const uint32_t dx = has_dx ? p.slot(bytes, kSlotOutput) : 0;
  const uint32_t dw = has_dw ? p.slot(mul_sat(extent, elem), kSlotOutput) : 0;
  const uint32_t db = has_db ? p.slot(mul_sat(extent, elem), kSlotOutput) : 0;
  if (extent == 0) return TILER_HIP_OK;
  if (extent > 0xffffffffull) return p.refuse(TILER_HIP_REFUSE_CAPACITY, "row longer than 2^32 - 1 elements");
  char name[64];
  const bool sums = has_dw || has_db;
  if (!has_dx && !sums) return TILER_HIP_OK;
  const uint64_t vec = 16 / elem, pieces = ceil_div(extent, vec);
  const uint32_t waves = pieces <= 64 ? 1 : pieces <= 128 ? 2 : pieces <= 256 ? 4 : pieces <= 512 ? 8 : 16;
  uint64_t count = 0;  // partials of dw's and db's sums
  uint32_t partials = 0;
  if (rows && extent >= vec && pieces <= 2048) {
    // Rows in registers, 8 / WAVES of them (or one of 16 waves) per workgroup at
    // a time, at most as many workgroups as run at once, so that there are few
    // partials.  Longer rows are streamed: 4096 x 12288 f32 341 us, 2048 x 18432
    // bf16 226.
    const uint64_t groups = waves == 16 ? rows : ceil_div(rows, 8 / waves);
    const uint64_t most = (waves == 16 ? 1ull : 2ull) * t.compute_units;
    count = groups < most ? groups : most;
    if (sums && count > 1) partials = p.slot(mul_sat(mul_sat(count, ceil_div(extent, 8) * 8), 8), kSlotScratch);
    std::snprintf(name, sizeof(name), "tiler_layer_norm_grad_%s_w%uc%u", type_name(dtype), waves,
                  pieces <= 1024 ? 1u : 2u);
    Launch& l = p.add(name, (uint32_t)count, 1, waves == 16 ? 1024 : 512).ptr(dy).ptr(x);
    slot_or_null(l, has_w, w);
    l.ptr(mean).ptr(rstd).u64(rows).u64(extent);
    slot_or_null(l, has_dx, dx);
    slot_or_null(l, sums && count > 1, partials);
    slot_or_null(l, has_dw, dw);
    slot_or_null(l, has_db, db);
    if (!sums || count == 1) return TILER_HIP_OK;
  } else if (rows) {
    if (has_dx) {
      std::snprintf(name, sizeof(name), "tiler_layer_norm_grad_%s_s", type_name(dtype));
      Launch& l = p.add(name, (uint32_t)(rows < kRowWorkgroups ? rows : kRowWorkgroups), 1, 256).ptr(dy).ptr(x);
      slot_or_null(l, has_w, w);
      l.ptr(mean).ptr(rstd).u64(rows).u64(extent).ptr(dx);
    }
    if (!sums) return TILER_HIP_OK;
    count = ceil_div(rows, 16) < t.compute_units ? ceil_div(rows, 16) : t.compute_units;
    partials = p.slot(mul_sat(mul_sat(count, ceil_div(extent, 8) * 8), 8), kSlotScratch);
    std::snprintf(name, sizeof(name), "tiler_layer_norm_columns_%s", type_name(dtype));
    p.add(name, column_groups(extent, 256), (uint32_t)count, 256)
        .ptr(dy).ptr(x).ptr(mean).ptr(rstd).u64(rows).u64(extent).u64(ceil_div(rows, count)).ptr(partials);
  } else if (!sums) {
    return TILER_HIP_OK;
  }
  std::snprintf(name, sizeof(name), "tiler_layer_norm_columns_final_%s", type_name(dtype));
  Launch& l = p.add(name, column_groups(extent, 64), 2, 1024);
  slot_or_null(l, count > 0, partials);  // no rows: zeros
  l.u32((uint32_t)count).u64(extent);
  slot_or_null(l, has_dw, dw);
  slot_or_null(l, has_db, db);
  return TILER_HIP_OK;
}

namespace {

tiler_hip_status check_product(uint64_t m, uint64_t n, uint64_t k, Program& p) {
  if (k == 0) return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "empty contracted extent");
  // a tile's rows lie within 32-bit offsets of its first: k below 2^24 elements
  if (m > 0x7fffff00ull || n > 0x7fffff00ull || k >= (1ull << 24) || ceil_div(m, 128) > 65535 ||
      !grid_holds(ceil_div(n, 64), 256))
    return p.refuse(TILER_HIP_REFUSE_CAPACITY, "contraction extents beyond the launch profile");
  return TILER_HIP_OK;
}

// The staged forms move 16-byte pieces of rows `row_bytes` apart and address a
// 256-row panel through one buffer resource (below 2^31 bytes).
bool staged_rows(uint64_t row_bytes) { return row_bytes % 16 == 0 && row_bytes * 256 < (1ull << 31); }

// A form of a staged product: a workgroup's rows and columns of the result, its
// threads, and what its run takes (us).  With W workgroups, q = ceil(W / CUs) and
// s slices of 128 bytes of depth:
//   kOne   one workgroup to a CU      c0 + q (c1 + c2 s)
//   kTwo   two workgroups to a CU     c0 + floor(q / 2) (c1 + c2 s) + (q mod 2) (c3 + c4 s)
//   kFew   a slice in eight a wave, t = ceil(s / 8)
//                                     c0 + q (c1 + c2 t) + c3 t + c4 t max(W / CUs, 1)
// The constants are least squares fits of measured times (m 1 .. 4096, n 600 ..
// 28672, k 800 .. 8192, at most 3000 workgroups): the form of the least estimate
// is 1% slower than the fastest in the mean.  Beyond those sizes they go on in
// rounds and slices as they are (int8 k = 14336 with its rows' quantization: 16 x
// 4096 14.7 us, 4.0 TB/s; 4096 x 4096 215, 2.2 P operations/s).
struct ProductForm {
  const char* name;
  uint32_t rows, cols, threads;
  enum Kind { kOne, kTwo, kFew } kind;
  double c[5];
};

// us, by size: 16 x 14336 x 4096 few1x1 45, t64_d 100; 301 of them t160_w 80, t192 90,
// t128 124; 4096 of them t256 740 (750 .. 767 on other cards), t128 830; 512 x 4096 x 4096 t128_d 39, t256_n 52.
constexpr ProductForm kGatedForms[] = {
    {"few1x1", 16, 16, 512, ProductForm::kFew, {2.591, 0.235, 0.356, 0.131, 0.151}},
    {"few2x1", 32, 16, 512, ProductForm::kFew, {2.524, 0.481, 0.610, 0, 0.115}},
    {"few4x1", 64, 16, 512, ProductForm::kFew, {1.224, 1.963, 0.888, 0, 0.142}},
    {"few4x2", 64, 32, 512, ProductForm::kFew, {1.264, 2.788, 1.431, 0, 0}},
    {"t64_d", 64, 64, 256, ProductForm::kOne, {1.747, 1.993, 0.351}},
    {"t96_d", 96, 64, 256, ProductForm::kOne, {1.914, 2.338, 0.435}},
    {"t128_d", 128, 64, 256, ProductForm::kOne, {1.567, 2.883, 0.511}},
    {"t96", 96, 64, 256, ProductForm::kTwo, {0.826, 2.393, 0.767, 1.920, 0.581}},
    {"t128", 128, 64, 256, ProductForm::kTwo, {1.502, 2.597, 0.915, 2.333, 0.611}},
    {"t192_n", 192, 64, 512, ProductForm::kOne, {1.186, 4.003, 0.623}},
    {"t256_n", 256, 64, 512, ProductForm::kOne, {0, 6.050, 0.756}},
    {"t160_w", 160, 128, 512, ProductForm::kOne, {0.029, 7.031, 0.923}},
    {"t192", 192, 128, 512, ProductForm::kOne, {0, 6.068, 1.019}},
    {"t256", 256, 128, 512, ProductForm::kOne, {0, 7.392, 1.237}},
};
// us, by size: 16 x 4096 x 4096 few1x1 6.2; 301 x 4096 x 4096 t64_d 15.6 (two slices in LDS 20.7);
// 4096 x 4096 x 4096 t256 59.4, t128 64.
constexpr ProductForm kInt8Forms[] = {
    {"few1x1", 16, 16, 512, ProductForm::kFew, {2.586, 0.193, 0.091, 0.172, 0.256}},
    {"few2x1", 32, 16, 512, ProductForm::kFew, {2.499, 0.363, 0.274, 0.052, 0.271}},
    {"few2x2", 32, 32, 512, ProductForm::kFew, {2.376, 0.655, 0.496, 0, 0.245}},
    {"few4x2", 64, 32, 512, ProductForm::kFew, {1.207, 2.072, 1.051, 0, 0.012}},
    {"few4x4", 64, 64, 512, ProductForm::kFew, {0.825, 3.623, 1.313, 0, 0.150}},
    {"t64_d", 64, 128, 256, ProductForm::kOne, {0.976, 2.979, 0.328}},
    {"t96_d", 96, 128, 256, ProductForm::kOne, {0.884, 3.723, 0.416}},
    {"t96", 96, 128, 256, ProductForm::kTwo, {0.821, 5.652, 0.613, 2.477, 0.535}},
    {"t128", 128, 128, 256, ProductForm::kTwo, {1.091, 6.483, 0.727, 2.924, 0.584}},
    {"t192", 192, 256, 512, ProductForm::kOne, {0, 7.540, 0.934}},
    {"t256", 256, 256, 512, ProductForm::kOne, {0, 9.259, 1.178}},
};

// A form's workgroups.  The few-row forms take their column panels eight at a
// time, one to an XCD.
uint64_t workgroups(const ProductForm& f, uint64_t m, uint64_t n) {
  const uint64_t rows = ceil_div(m, f.rows), cols = ceil_div(n, f.cols);
  return mul_sat(rows, f.kind == ProductForm::kFew && cols >= 8 ? ceil_div(cols, 8) * 8 : cols);
}

// q rounds of workgroups (`share` of the CUs, kFew's) with s slices each.
double estimate(const ProductForm& f, double q, double s, double share) {
  if (f.kind == ProductForm::kOne) return f.c[0] + q * (f.c[1] + f.c[2] * s);
  if (f.kind == ProductForm::kTwo) {
    const double pairs = std::floor(q / 2);
    return f.c[0] + pairs * (f.c[1] + f.c[2] * s) + (q - 2 * pairs) * (f.c[3] + f.c[4] * s);
  }
  const double part = std::ceil(s / 8);
  return f.c[0] + q * (f.c[1] + f.c[2] * part) + f.c[3] * part + f.c[4] * part * (share > 1 ? share : 1);
}

// The form of the least estimate, or null where no form's grid fits a launch.
template <size_t N>
const ProductForm* choose(const ProductForm (&forms)[N], const Target& t, uint64_t m, uint64_t n, uint64_t slices) {
  const ProductForm* best = nullptr;
  double least = 0;
  for (const ProductForm& f : forms) {
    const uint64_t w = workgroups(f, m, n);
    if (!grid_holds(w, f.threads)) continue;
    const double us = estimate(f, (double)ceil_div(w, t.compute_units), (double)slices, (double)w / t.compute_units);
    if (!best || us < least) best = &f, least = us;
  }
  return best;
}

// Rows of the guarded forms' tiles, 64 or 128: 64 where those are at most one to
// a CU, or no more of them.  us, 64 and 128: int8 257 x 5001 x 1111 15.0 / 23.4,
// 2048 x 4096 x 4095 86 / 70; gated 200 x 4096 x 4095 48 / 66, 777 of them 125 / 99.
uint32_t guarded_rows(const Target& t, uint64_t m, uint64_t column_tiles) {
  return m <= 64 || mul_sat(ceil_div(m, 64), column_tiles) <= t.compute_units ? 64 : 128;
}

// The gradients' products: a form's tile, the depth split over `splits` workgroups a
// tile where the tiles alone leave CUs idle, the binary32 partials added by one
// more launch.  The least of the same estimates, with the results' stores (a
// million elements: 0.39 us) or the partials' (1.31 a part, 1.55 and 0.29 a part
// besides): fits of 1031 times of sizes spread over m 1 .. 4096, n to 10424, k to
// 4096, 1.6% slower than the fastest form in the mean.  us, dx of 2048 x 8192 x
// 2048: t256 in four 135, t128 in two 159, t256 whole 316; of 7 x 2048 x 872 t64_d
// in eight 11.3, t128 in 32 16.3; the weights' gradients of 8192 x 512 x 512: t64_d
// in four 24, t128 whole 78; of 777 x 1365 x 509: t64_d 10.9, t128 13.1.
constexpr ProductForm kGradientForms[] = {
    {"t64_d", 64, 128, 256, ProductForm::kOne, {2.974, 1.401, 0.395}},
    {"t128", 128, 128, 256, ProductForm::kTwo, {4.210, 0, 0.900, 0.225, 0.588}},
    {"t256", 256, 256, 512, ProductForm::kOne, {6.412, 0.164, 1.179}},
};
struct GradientChoice {
  const ProductForm* form = nullptr;
  uint32_t splits = 1;
  uint64_t tiles = 0;
};
GradientChoice choose_gradient(const Target& t, uint64_t halves, uint64_t rows, uint64_t cols, uint64_t slices) {
  GradientChoice best;
  double least = 0;
  const double results = (double)halves * (double)rows * (double)cols * 1e-6;
  for (const ProductForm& f : kGradientForms) {
    const uint64_t tiles = mul_sat(halves * ceil_div(rows, f.rows), ceil_div(cols, f.cols));
    if (!grid_holds(tiles, 512)) continue;
    for (uint32_t splits = 1; splits <= 32 && (splits == 1 || splits * 2 <= slices); ++splits) {
      const double q = std::ceil((double)tiles * splits / t.compute_units);
      double us = estimate(f, q, (double)ceil_div(slices, splits), 0);
      us += splits > 1 ? 1.546 + splits * (0.294 + 1.309 * results) : 0.386 * results;
      if (!best.form || us < least) best = {&f, splits, tiles}, least = us;
    }
  }
  return best;
}

Launch& add_gradient(Program& p, const char* stem, const GradientChoice& c) {
  const std::string name = std::string(stem) + "_" + c.form->name;
  return p.add(name.c_str(), (uint32_t)c.tiles, c.splits, c.form->threads);
}

}  // namespace

// Slots: x, wg, wu, h, [gate, up].
tiler_hip_status plan_gated_contract_bf16(const Target& t, uint32_t parts, uint64_t m, uint64_t n, uint64_t k,
                                          const uintptr_t* addr, Program& p) {
  if (parts & ~(uint32_t)TILER_HIP_GATED_KEEP) return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "gated_contract parts");
  const bool keep = parts & TILER_HIP_GATED_KEEP;
  const uint64_t out = mul_sat(mul_sat(m, n), 2), weight = mul_sat(mul_sat(n, k), 2);
  const uint32_t x = p.slot(mul_sat(mul_sat(m, k), 2), kSlotInput);
  const uint32_t wg = p.slot(weight, kSlotInput), wu = p.slot(weight, kSlotInput);
  const uint32_t h = p.slot(out, kSlotOutput);
  const uint32_t gate = keep ? p.slot(out, kSlotOutput) : 0, up = keep ? p.slot(out, kSlotOutput) : 0;
  if (tiler_hip_status st = check_product(m, n, k, p); st != TILER_HIP_OK) return st;
  if (m == 0 || n == 0) return TILER_HIP_OK;
  const bool al = staged_rows(2 * k) && aligned16(addr[x]) && aligned16(addr[wg]) && aligned16(addr[wu]);
  const ProductForm* const f = al ? choose(kGatedForms, t, m, n, ceil_div(k, 64)) : nullptr;
  const uint32_t rows = guarded_rows(t, m, ceil_div(n, 64));
  const std::string name = "tiler_gated_bf16_" + (f ? std::string(f->name) : "g" + std::to_string(rows));
  Launch& l = (f ? p.add(name.c_str(), (uint32_t)workgroups(*f, m, n), 1, f->threads)
                 : p.add(name.c_str(), (uint32_t)ceil_div(n, 64), (uint32_t)ceil_div(m, rows), 256))
                  .ptr(x).ptr(wg).ptr(wu).u32((uint32_t)m).u32((uint32_t)n).u32((uint32_t)k).ptr(h);
  slot_or_null(l, keep, gate);
  slot_or_null(l, keep, up);
  return TILER_HIP_OK;
}

// Slots: x, wg, wu, gate, up, dh, [dx,] [dwg, dwu,] and scratch: dG with dU
// behind it, copies of x and of the weights where their rows do not start on 16
// bytes, partial sums of dx.
tiler_hip_status plan_gated_contract_bf16_backward(const Target& t, uint32_t parts, uint64_t m, uint64_t n, uint64_t k,
                                                   const uintptr_t* addr, Program& p) {
  if (parts & ~(uint32_t)(TILER_HIP_GATED_DX | TILER_HIP_GATED_DW))
    return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "gated_contract_backward parts");
  const bool has_dx = parts & TILER_HIP_GATED_DX, has_dw = parts & TILER_HIP_GATED_DW;
  const uint64_t mid = mul_sat(mul_sat(m, n), 2), weight = mul_sat(mul_sat(n, k), 2), in = mul_sat(mul_sat(m, k), 2);
  const uint32_t x = p.slot(in, kSlotInput), wg = p.slot(weight, kSlotInput), wu = p.slot(weight, kSlotInput);
  const uint32_t gate = p.slot(mid, kSlotInput), up = p.slot(mid, kSlotInput), dh = p.slot(mid, kSlotInput);
  const uint32_t dx = has_dx ? p.slot(in, kSlotOutput) : 0;
  const uint32_t dwg = has_dw ? p.slot(weight, kSlotOutput) : 0, dwu = has_dw ? p.slot(weight, kSlotOutput) : 0;
  if (tiler_hip_status st = check_product(m, n, k, p); st != TILER_HIP_OK) return st;
  if (n > (1ull << 22) - 64 || k > (1ull << 22) - 64)  // 256 of their rows lie within one buffer resource
    return p.refuse(TILER_HIP_REFUSE_CAPACITY, "contraction extents beyond the launch profile");
  if (!parts) return TILER_HIP_OK;
  const uint64_t ld = ceil_div(n, 64) * 64, ldk = ceil_div(k, 8) * 8;
  const uint32_t dg = p.slot(mul_sat(mul_sat(m, ld), 4), kSlotScratch);
  const uint32_t m32 = (uint32_t)m, n32 = (uint32_t)n, k32 = (uint32_t)k;
  // The products run over n and over m: nothing of the operands is read where either is 0.
  const bool copy_w = has_dx && m && n && !(k % 8 == 0 && aligned16(addr[wg]) && aligned16(addr[wu]));
  const bool copy_x = has_dw && m && n && !(k % 8 == 0 && aligned16(addr[x]));
  const uint32_t to_x = copy_x ? p.slot(mul_sat(mul_sat(m, ldk), 2), kSlotScratch) : 0;
  const uint32_t to_w = copy_w ? p.slot(mul_sat(mul_sat(n, ldk), 4), kSlotScratch) : 0;
  if (m && n) {
    // workgroups that form dG and dU, then those that copy: at most 8192 of each
    auto groups = [](uint64_t pieces) { return pieces < 8192 * 256ull ? ceil_div(pieces, 256) : 8192; };
    const uint64_t copies = ((copy_x ? m : 0) + (copy_w ? 2 * n : 0)) * (ldk / 8);
    const uint32_t forming = (uint32_t)groups(m * (ld / 8));
    Launch& l = p.add("tiler_gated_bf16_grad", forming + (uint32_t)groups(copies), 1, 256)
                    .ptr(gate).ptr(up).ptr(dh).ptr(x).ptr(wg).ptr(wu).u32(m32).u32(n32).u32(k32).u32(forming).ptr(dg);
    slot_or_null(l, copy_x, to_x);
    slot_or_null(l, copy_w, to_w);
  }
  const GradientChoice fx = choose_gradient(t, 1, m, k, n ? 2 * (ld / 64) : 0), fw = choose_gradient(t, 2, n, k, ceil_div(m, 64));
  if ((has_dx && m && !fx.form) || (has_dw && n && !fw.form))
    return p.refuse(TILER_HIP_REFUSE_CAPACITY, "contraction extents beyond the launch profile");
  const bool sum_x = has_dx && m && fx.splits > 1, sum_w = has_dw && n && fw.splits > 1;
  const uint32_t of_x = sum_x ? p.slot(mul_sat(mul_sat(fx.splits, m * k), 4), kSlotScratch) : 0;
  const uint32_t of_w = sum_w ? p.slot(mul_sat(mul_sat(fw.splits, n * k), 8), kSlotScratch) : 0;
  if (has_dx && m) {
    Launch& l = add_gradient(p, "tiler_gated_bf16_dx", fx).ptr(dg).ptr(copy_w ? to_w : wg);
    slot_or_null(l, !copy_w, wu);
    l.u32((uint32_t)(copy_w ? ldk : k)).u32(m32).u32(n32).u32(k32).ptr(dx).u32(fx.splits);
    slot_or_null(l, sum_x, of_x);
  }
  if (has_dw && n) {
    Launch& l = add_gradient(p, "tiler_gated_bf16_dw", fw)
                    .ptr(dg).ptr(copy_x ? to_x : x).u32((uint32_t)(copy_x ? ldk : k)).u32(m32).u32(n32).u32(k32)
                    .ptr(dwg).ptr(dwu).u32(fw.splits);
    slot_or_null(l, sum_w, of_w);
  }
  if (sum_x || sum_w) {
    const uint64_t pieces = (sum_x ? ceil_div(m * k, 4) : 0) + (sum_w ? 2 * ceil_div(n * k, 4) : 0);
    const uint64_t groups = ceil_div(pieces, 256);
    Launch& l = p.add("tiler_gated_bf16_sum", (uint32_t)(groups < 8192 ? groups : 8192), 1, 256);
    slot_or_null(l, sum_x, of_x);
    l.u32(fx.splits).u64(sum_x ? m * k : 0);
    slot_or_null(l, sum_x, dx);
    slot_or_null(l, sum_w, of_w);
    l.u32(fw.splits).u64(sum_w ? n * k : 0);
    slot_or_null(l, sum_w, dwg);
    slot_or_null(l, sum_w, dwu);
  }
  return TILER_HIP_OK;
}

// Slots: x, q, scales.
tiler_hip_status plan_quantize_rows_i8(const Target& t, uint32_t dtype, uint64_t rows, uint64_t extent, const uintptr_t*,
                                       Program& p) {
  if (dtype != TILER_HIP_F32 && dtype != TILER_HIP_BF16)
    return p.refuse(TILER_HIP_REFUSE_UNSUPPORTED, "quantize_rows dtype");
  const uint64_t n = mul_sat(rows, extent);
  const uint32_t x = p.slot(mul_sat(n, dtype == TILER_HIP_BF16 ? 2 : 4), kSlotInput);
  const uint32_t q = p.slot(n, kSlotOutput), scales = p.slot(mul_sat(rows, 4), kSlotOutput);
  if (rows == 0) return TILER_HIP_OK;
  if (extent == 0) return p.refuse(TILER_HIP_REFUSE_INVALID_ARGUMENT, "rows without elements have no scale");
  if (extent > 0xffffffffull) return p.refuse(TILER_HIP_REFUSE_CAPACITY, "row longer than 2^32 - 1 elements");
  char name[64];
  const RowForm f = row_form(t, rows, extent, dtype == TILER_HIP_BF16 ? 8 : 4, dtype == TILER_HIP_BF16 ? 2 : 4);
  std::snprintf(name, sizeof(name), "tiler_quantize_rows_i8_%s_%s", type_name(dtype), f.name);
  p.add(name, (uint32_t)f.grid, 1, f.block)
      .ptr(x).u64(rows).u64(extent).ptr(q).ptr(scales);
  return TILER_HIP_OK;
}

// Slots: a, b, a_scales, b_scales, c.
tiler_hip_status plan_contract_i8(const Target& t, uint32_t out_dtype, uint64_t m, uint64_t n, uint64_t k,
                                  const uintptr_t* addr, Program& p) {
  if (out_dtype != TILER_HIP_F32 && out_dtype != TILER_HIP_BF16)
    return p.refuse(TILER_HIP_REFUSE_UNSUPPORTED, "contract_i8 result dtype");
  const uint32_t a = p.slot(mul_sat(m, k), kSlotInput), b = p.slot(mul_sat(n, k), kSlotInput);
  const uint32_t sa = p.slot(mul_sat(m, 4), kSlotInput), sb = p.slot(mul_sat(n, 4), kSlotInput);
  const uint32_t c = p.slot(mul_sat(mul_sat(m, n), out_dtype == TILER_HIP_BF16 ? 2 : 4), kSlotOutput);
  if (tiler_hip_status st = check_product(m, n, k, p); st != TILER_HIP_OK) return st;
  if (k > 131071) return p.refuse(TILER_HIP_REFUSE_CAPACITY, "a sum of more than 131071 products could leave 32 bits");
  if (m == 0 || n == 0) return TILER_HIP_OK;
  const bool al = staged_rows(k) && aligned16(addr[a]) && aligned16(addr[b]);
  const ProductForm* const f = al ? choose(kInt8Forms, t, m, n, ceil_div(k, 128)) : nullptr;
  const uint32_t rows = guarded_rows(t, m, ceil_div(n, 128));
  const std::string name = std::string("tiler_contract_i8_") + type_name(out_dtype) + "_" +
                           (f ? std::string(f->name) : "g" + std::to_string(rows));
  (f ? p.add(name.c_str(), (uint32_t)workgroups(*f, m, n), 1, f->threads)
     : p.add(name.c_str(), (uint32_t)ceil_div(n, 128), (uint32_t)ceil_div(m, rows), 256))
      .ptr(a).ptr(b).ptr(sa).ptr(sb).u32((uint32_t)m).u32((uint32_t)n).u32((uint32_t)k).ptr(c);
  return TILER_HIP_OK;
}

}  // namespace tiler_rt
