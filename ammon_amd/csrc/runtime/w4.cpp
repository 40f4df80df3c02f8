// w4.cpp -- C-ABI entry points of the 4-bit weights (AMMON_W4) and the rows of 8-bit digits
// (AMMON_Q8, AMMON_Q24): validate, pick the variant, launch.  No counterpart in the reference.
#include <hip/hip_runtime_api.h>

#include <cstring>

#include "ops_common.h"

using namespace ammon_rt;

namespace {

// A launch has fewer than 2^32 work items in a dimension.
constexpr uint64_t kMaxWorkgroups = (1ull << 32) / kWorkgroup - 1;

bool valid_digits(ammon_dtype d) { return d == AMMON_Q8 || d == AMMON_Q24; }

ammon_status shape_check(const char *what, uint32_t rows, uint32_t n) {
  AMMON_CHECK(rows > 0 && n > 0, "%s: empty shape (%u rows of %u)", what, rows, n);
  AMMON_CHECK(cdiv(rows, 16) <= kMaxWorkgroups, "%s: %u rows are too many", what, rows);
  AMMON_CHECK(n < (1u << 22), "%s: rows of %u numbers are too long", what, n);
  return AMMON_OK;
}

ammon_status aligned(const char *what, const void *p, const char *name) {
  AMMON_CHECK(((uintptr_t)p & 15u) == 0, "%s: %s must be 16-byte aligned", what, name);
  return AMMON_OK;
}

#define TRY(expr)                         \
  do {                                    \
    const ammon_status st_ = (expr);      \
    if (st_ != AMMON_OK) return st_;      \
  } while (0)

// Panels of 16 rows: queries, keys and values begin one each.
ammon_status qkv_check(const char *what, uint64_t q_dim, uint64_t kv_dim) {
  AMMON_CHECK(q_dim % 16 == 0 && kv_dim % 16 == 0,
              "%s: W4 queries, keys and values must be a multiple of 16 rows each", what);
  return AMMON_OK;
}

// ---- prompt products -------------------------------------------------------------------------
struct W4GemmArgs {
  int mode;
  const void *w0, *w1, *w2;
  uint32_t d, n, rows, tokens;
  const void *x;
  ammon_dtype x_dtype;
  const float *residual;
  float *y;
  size_t y_bytes;
  void *k_cache, *v_cache;
  size_t kv_bytes;
  const ammon_decode_step *step;
  const float *table;
  uint32_t kv_dim, head, seq;
  ammon_dtype kv_dtype;
  bool kv_rows;
  void *ws;
  size_t ws_bytes;
};

ammon_status w4_gemm(ammon_runtime *rt, ammon_stream stream, const W4GemmArgs &a, const char *what) {
  AMMON_CHECK(a.w0 && a.x && a.y, "%s: NULL weight, x or y", what);
  AMMON_CHECK(valid_digits(a.x_dtype), "%s: x is rows of digits (AMMON_Q8 or AMMON_Q24), not dtype %d",
              what, (int)a.x_dtype);
  TRY(shape_check(what, a.rows, a.n));
  AMMON_CHECK(a.d > 0 && a.rows < (1u << 31), "%s: empty or too large (d=%u)", what, a.d);
  TRY(shape_check(what, a.tokens, a.n));
  const void *const ws[] = {a.w0, a.w1, a.w2};
  const uint32_t wd[] = {a.d, a.mode == AMMON_GEMV_QKV ? a.kv_dim : a.d, a.kv_dim};
  for (int i = 0; i < 3; ++i)
    if (ws[i]) {
      TRY(aligned(what, ws[i], "weights"));
      AMMON_CHECK(!overlaps(ws[i], ammon_w4_bytes(wd[i], a.n), a.y, a.y_bytes), "%s: y overlaps weights", what);
    }
  TRY(aligned(what, a.x, "x"));
  const size_t xbytes = ammon_q8_bytes(a.x_dtype, a.tokens, a.n);
  AMMON_CHECK(!overlaps(a.x, xbytes, a.y, a.y_bytes), "%s: y overlaps x", what);
  AMMON_CHECK(!a.residual || a.residual == a.y || !overlaps(a.residual, a.y_bytes, a.y, a.y_bytes),
              "%s: residual partially overlaps y", what);
  for (const void *to : {a.k_cache, a.v_cache})
    AMMON_CHECK(!to || (!overlaps(to, a.kv_bytes, a.x, xbytes) && !overlaps(to, a.kv_bytes, a.y, a.y_bytes)),
                "%s: k or v overlaps x or q", what);
  if (a.ws) {
    TRY(aligned(what, a.ws, "workspace"));
    AMMON_CHECK(!overlaps(a.ws, a.ws_bytes, a.x, xbytes) && !overlaps(a.ws, a.ws_bytes, a.y, a.y_bytes) &&
                    !(a.residual && overlaps(a.ws, a.ws_bytes, a.residual, a.y_bytes)) &&
                    !(a.k_cache && overlaps(a.ws, a.ws_bytes, a.k_cache, a.kv_bytes)) &&
                    !(a.v_cache && overlaps(a.ws, a.ws_bytes, a.v_cache, a.kv_bytes)),
                "%s: workspace overlaps x, y, residual, k or v", what);
  }
  ammon_k_gemm p = {};
  p.w0 = a.w0;
  p.w1 = a.w1;
  p.w2 = a.w2;
  p.x = (const float *)a.x;
  p.residual = a.residual;
  p.y = a.y;
  p.k_cache = a.k_cache;
  p.v_cache = a.v_cache;
  p.step = (const ammon_k_step *)a.step;
  p.table = a.table;
  p.d = a.d;
  p.n = a.n;
  p.rows = a.rows;
  p.tokens = a.tokens;
  p.kv_dim = a.kv_dim;
  p.head = a.head;
  p.seq = a.seq;
  p.kv_dtype = (uint32_t)a.kv_dtype;
  p.kv_rows = a.kv_rows;
  const bool gated = a.mode == AMMON_GEMV_SWIGLU, q24 = a.x_dtype == AMMON_Q24;
  const uint64_t panels = cdiv(gated ? a.d : a.rows, 16);
  // Of the tiles, the big ones optionally with the reduction split into 2, 4 or 8 ranges (a
  // workspace, no SwiGLU), the one with the least estimated time, in us: a launch takes 3.5 (of
  // sixteen waves 3.85); a group of 128 takes a CU's first workgroup `first` and each further one
  // `more` (the big ones, of which several take turns, `more` each as soon as there are two); a
  // split adds a second launch and the sums' traffic.  Fitted to 4096 x 4096, 6144 x 4096, 4096 x
  // 14336, 10240 x 8192, 8192 x 28672, 5003 x 2080, 1024 x 8192, 128256 x 4096, 288 x 288 and
  // (SwiGLU) 28672 x 4096, 11264 x 2048 and 57344 x 8192, 1 to 2048 tokens, both digit types.  Of 300
  // such products, every tile and split timed, the one so chosen is 1.3% slower than the best on
  // average, more than 10% in eight, at most 58% (1024 x 8192, 301 tokens of Q8: 64-token tiles in
  // eight ranges 20.7 us, 32-token tiles 13.0; the next worst 22%).  E.g. of 6144 x 4096, 41 tokens
  // of Q24: 16-token tiles 16.1 us, of two panels 13.2, of four 12.6 (estimate 13.5), long tiles in
  // eight ranges 14.3, whole 50.8.
  const uint32_t groups = cdiv(a.n, 128), cus = (uint32_t)std::max(rt->info.compute_units, 1);
  const W4Tile *const tiles = kW4Tile[q24], *tile = nullptr;
  uint32_t ksplit = 1, per = 1;  // per: panels of results per workgroup
  double best = 1e300;
  for (int i = 0; i < kW4Tiles; ++i) {
    const W4Tile *t = &tiles[i];
    const bool big = t->big;
    if ((gated && t->first_gated == 0) || (rt->w4_tile[q24] >= 0 && rt->w4_tile[q24] != i)) continue;
    const uint32_t pp = big && gated ? t->panels / 2 : t->panels;
    for (uint32_t k = 1; k <= 8; k *= 2) {
      const uint64_t sums = (uint64_t)k * a.tokens * a.rows * 4;
      if (k > 1 && (!big || gated || !a.ws || sums > a.ws_bytes || sums > (64ull << 20) || groups < 4 * k)) break;
      if (rt->w4_ranges && k != rt->w4_ranges) continue;
      // (the XCDs get row blocks' ranges in turn)
      const uint64_t wgs = (uint64_t)cdiv((uint64_t)cdiv(panels, pp) * k, 8) * 8 * cdiv(a.tokens, t->tokens);
      const uint64_t turns = (wgs + cus - 1) / cus;
      const double first = gated ? t->first_gated : t->first, more = gated ? t->more_gated : t->more;
      const double group = big ? (turns > 1 ? (double)turns * more : first) : first + (double)(turns - 1) * more;
      const double us = (t->waves == 16 ? 3.85 : 3.5) + cdiv(groups, k) * group + (k > 1 ? 2.5 + sums / 4e6 : 0);
      if (us < best) best = us, tile = t, ksplit = k, per = pp;
    }
  }
  AMMON_CHECK(tile, "%s: the tile chosen does not take this call", what);
  if (ksplit > 1) {
    p.ws = (float *)a.ws;
    p.ksplit = ksplit;
    p.kchunks = cdiv(groups, ksplit);
  }
  const uint64_t grid = (uint64_t)cdiv((uint64_t)cdiv(panels, per) * ksplit, 8) * 8 * cdiv(a.tokens, tile->tokens);
  AMMON_CHECK(grid * (tile->waves / 4) <= kMaxWorkgroups, "%s: grid too large", what);
  VALIDATE_ONLY();
  DeviceGuard guard(rt->device);
  void *args[] = {&p};
  const hipError_t e = hipModuleLaunchKernel(rt->k.w4_gemm[q24][tile - tiles][a.mode], (uint32_t)grid, 1, 1,
                                             64 * tile->waves, 1, 1, 0,
                                             stream ? (hipStream_t)stream : rt->stream, args, nullptr);
  if (e != hipSuccess) return hip_error(e, what);
  if (ksplit == 1) return AMMON_OK;
  // the ranges' sums (QKV: per row pair, then the rotation and stores)
  const bool pairs = a.mode == AMMON_GEMV_QKV;
  const uint64_t elems = (uint64_t)a.tokens * (pairs ? a.rows / 2 : a.d);
  return launch(rt, stream, pairs ? rt->k.gemm_reduce_qkv : rt->k.gemm_reduce,
                (uint32_t)std::min<uint64_t>((elems + kWorkgroup - 1) / kWorkgroup, cus * 4ull), 1, 0, p, what);
}

ammon_status w4_qkv(ammon_runtime *rt, ammon_stream stream, const void *x, ammon_dtype x_dtype,
                    uint32_t tokens, const void *wq, const void *wk, const void *wv, uint32_t dim,
                    uint32_t q_heads, uint32_t kv_heads, uint32_t head, float *q, void *k, void *v,
                    ammon_dtype kv_dtype, bool rows, uint32_t seq, const ammon_decode_step *step,
                    const float *table, void *workspace, size_t workspace_bytes, const char *what) {
  AMMON_CHECK(wq && wk && wv, "%s: NULL wq, wk or wv", what);
  AMMON_CHECK(k && v && step && table, "%s: NULL %s, step or table", what, rows ? "row buffer" : "cache");
  AMMON_CHECK(kv_dtype != AMMON_KV4, "%s: a KV4 cache takes rows (prefill_qkv_rope_w4, then kv4_store)", what);
  AMMON_CHECK(valid_dtype(kv_dtype), "%s: unknown kv dtype %d", what, (int)kv_dtype);
  AMMON_CHECK(q_heads > 0 && kv_heads > 0 && seq > 0, "%s: empty shape", what);
  AMMON_CHECK(head >= 2 && head % 2 == 0, "%s: head size %u must be even", what, head);
  const uint64_t q_dim = (uint64_t)q_heads * head, kv_dim = (uint64_t)kv_heads * head;
  TRY(qkv_check(what, q_dim, kv_dim));
  AMMON_CHECK(kv_dim <= q_dim, "%s: kv width must be no wider than q", what);
  AMMON_CHECK(q_dim + 2 * kv_dim < (1ull << 31), "%s: too many rows", what);
  const size_t kv_bytes = (size_t)kv_dim * (rows ? tokens : seq) * dsize(kv_dtype);
  AMMON_CHECK(!overlaps(k, kv_bytes, v, kv_bytes), "%s: key and value %s overlap", what,
              rows ? "rows" : "caches");
  AMMON_CHECK((((uintptr_t)k | (uintptr_t)v) & (kv_dtype == AMMON_BF16 ? 3u : 7u)) == 0,
              "%s: k and v must be aligned to pairs of numbers", what);
  W4GemmArgs a = {};
  a.mode = AMMON_GEMV_QKV;
  a.w0 = wq;
  a.w1 = wk;
  a.w2 = wv;
  a.d = (uint32_t)q_dim;
  a.n = dim;
  a.rows = (uint32_t)(q_dim + 2 * kv_dim);
  a.tokens = tokens;
  a.x = x;
  a.x_dtype = x_dtype;
  a.y = q;
  a.y_bytes = (size_t)tokens * q_dim * 4;
  a.k_cache = k;
  a.v_cache = v;
  a.kv_bytes = kv_bytes;
  a.step = step;
  a.table = table;
  a.kv_dim = (uint32_t)kv_dim;
  a.head = head;
  a.seq = seq;
  a.kv_dtype = kv_dtype;
  a.kv_rows = rows;
  a.ws = workspace;
  a.ws_bytes = workspace ? workspace_bytes : 0;
  return w4_gemm(rt, stream, a, what);
}

// Rows x (+ residual, normalised with w) into digits.
ammon_status q8_rows(ammon_runtime *rt, ammon_stream stream, const float *x, const float *residual,
                     float *sum, const void *w, ammon_dtype w_dtype, float eps, uint32_t tokens, uint32_t n,
                     void *out, ammon_dtype dtype, const char *what) {
  AMMON_CHECK(x && out, "%s: NULL x or rows", what);
  AMMON_CHECK(valid_digits(dtype), "%s: rows are AMMON_Q8 or AMMON_Q24, not dtype %d", what, (int)dtype);
  TRY(shape_check(what, tokens, n));
  AMMON_CHECK(tokens <= kMaxWorkgroups / 2 - 128, "%s: %u tokens are too many", what, tokens);
  TRY(aligned(what, out, "rows"));
  const size_t bytes = (size_t)tokens * n * 4, to = ammon_q8_bytes(dtype, tokens, n);
  AMMON_CHECK(!overlaps(x, bytes, out, to) && !(residual && overlaps(residual, bytes, out, to)) &&
                  !(sum && overlaps(sum, bytes, out, to)),
              "%s: rows overlap x, residual or sum", what);
  if (residual)
    for (const float *from : {x, residual})
      AMMON_CHECK(sum == from || !overlaps(sum, bytes, from, bytes), "%s: sum partially overlaps x or residual",
                  what);
  if (w) {
    const size_t wbytes = n * dsize(w_dtype);
    AMMON_CHECK(!overlaps(w, wbytes, out, to) && !(sum && overlaps(w, wbytes, sum, bytes)),
                "%s: weight overlaps rows or sum", what);
  }
  VALIDATE_ONLY();
  ammon_k_q8 p = {};
  p.x = x;
  p.residual = residual;
  p.sum = sum;
  p.w = w;
  p.rows = out;
  p.tokens = tokens;
  p.n = n;
  p.w_dtype = (uint32_t)w_dtype;
  p.eps = eps;
  // (a workgroup a token, of whole panels for each of the eight XCDs)
  DeviceGuard guard(rt->device);
  void *args[] = {&p};
  const hipError_t e = hipModuleLaunchKernel(
      rt->k.q8_rows[dtype == AMMON_Q24][n <= 4096 ? 0 : n <= 8192 ? 1 : 2], cdiv(tokens, 128) * 128, 1, 1,
      2 * kWorkgroup, 1, 1, 0, stream ? (hipStream_t)stream : rt->stream, args, nullptr);
  if (e != hipSuccess) return hip_error(e, what);
  return AMMON_OK;
}

}  // namespace

namespace ammon_rt {

const W4Tile kW4Tile[2][kW4Tiles] = {{{"t16", 1, 16, 8, 0.039, 0.044, 0.082, 0.081, false},
                                      {"t16_deep", 1, 16, 16, 0.035, 0.049, 0, 0, false},
                                      {"t16_x4", 4, 16, 8, 0.118, 0.112, 0.312, 0.254, false},
                                      {"t32_x2", 2, 32, 8, 0.094, 0.088, 0.207, 0.166, false},
                                      {"t64", 8, 64, 4, 0.48, 0.377, 0.48, 0.377, true},
                                      {"long", 8, 128, 4, 0.99, 0.693, 0.99, 0.693, true}},
                                     {{"t16", 1, 16, 8, 0.070, 0.089, 0.127, 0.126, false},
                                      {"t16_deep", 1, 16, 16, 0.066, 0.093, 0, 0, false},
                                      {"t16_x2", 2, 16, 8, 0.106, 0.110, 0.210, 0.181, false},
                                      {"t16_x4", 4, 16, 8, 0.163, 0.156, 0.361, 0.329, false},
                                      {"t64", 8, 64, 4, 0.93, 0.83, 0.93, 0.83, true},
                                      {"long", 16, 64, 4, 1.55, 1.44, 1.55, 1.44, true}}};
const char *const kW4WayName[kW4Ways] = {"k8_one", "k8", "k2", "k8_wide", "flat"};

ammon_status w4_gemv(ammon_runtime *rt, ammon_stream stream, const GemvArgs &a, const char *what,
                     uint32_t *grid_out) {
  AMMON_CHECK(a.w0 && a.x && a.y, "%s: NULL weight, x or y", what);
  TRY(shape_check(what, a.rows, a.n));
  AMMON_CHECK(a.d > 0, "%s: empty matrix (d=%u)", what, a.d);
  // (of the plain products gemv_at_position alone has a step, whose row of y it writes)
  AMMON_CHECK(a.mode != AMMON_GEMV_PLAIN || !a.step, "%s: takes no W4 weights", what);
  AMMON_CHECK(!a.norm_w || valid_dtype(a.norm_dtype), "%s: unknown norm dtype", what);
  AMMON_CHECK(!a.norm_w || (std::isfinite(a.eps) && a.eps >= 0.f), "%s: eps must be finite and >= 0", what);
  for (const void *w : {a.w0, a.w1, a.w2})
    if (w) TRY(aligned(what, w, "W4 weights"));
  const size_t ybytes = (size_t)a.d * 4;
  AMMON_CHECK(!overlaps(a.x, (size_t)a.n * 4, a.y, ybytes), "%s: y overlaps x", what);
  AMMON_CHECK(!a.residual || !overlaps(a.x, (size_t)a.n * 4, a.residual, ybytes), "%s: residual overlaps x", what);
  if (a.mode == AMMON_GEMV_QKV) TRY(qkv_check(what, a.d, a.kv_dim));
  // x's digits and scales, whole rounds of a set's chunks
  auto lds_of = [&](uint32_t ks) {
    const uint32_t round = ks * AMMON_W4_CHUNK;
    return (size_t)cdiv(cdiv(a.n, 128), round) * round * (4 * 128 + 16);
  };
  AMMON_CHECK(lds_of(8) + 4096 <= (size_t)rt->info.max_shared_per_block,
              "%s: reduction length n=%u needs %zu bytes of LDS; the device allows %d", what, a.n,
              lds_of(8) + 4096, rt->info.max_shared_per_block);
  ammon_k_gemv p = {};
  p.w0 = a.w0;
  p.w1 = a.w1;
  p.w2 = a.w2;
  p.x = a.x;
  p.norm_w = a.norm_w;
  p.residual = a.residual;
  p.y = a.y;
  p.k_cache = a.k_cache;
  p.v_cache = a.v_cache;
  p.step = (const ammon_k_step *)a.step;
  p.table = a.table;
  p.d = a.d;
  p.n = a.n;
  p.rows = a.rows;
  p.row_blocks = cdiv(a.rows, 16);
  p.norm_dtype = (uint32_t)a.norm_dtype;
  p.eps = a.eps;
  p.kv_dim = a.kv_dim;
  p.head = a.head;
  p.seq = a.seq;
  p.kv_dtype = (uint32_t)a.kv_dtype;
  p.kv_rows = a.kv_rows;
  p.cand_v = a.cand_v;
  p.cand_i = a.cand_i;
  // Where a CU has between 64 and 384 groups (14336 x 4096 twice, 224: 12.3 us, as sets 14.4; 10240 x
  // 8192, 160: 10.4 and 14.7; 4096 x 14336, 112: 8.4 and 9.6), its waves take them side by side.  With
  // fewer the sixteen waves' own costs show (4096 x 4096, 32: 5.0 and 3.7; 6144 x 4096, 48: 5.3 and
  // 4.8), with more the sets' order of reading, one panel after the other on the whole device (57344
  // x 8192, 896: 41.8 and 38.4; 8192 x 28672, 448: 22.4 and 22.1).
  // Sets of 8 waves, in workgroups of one, two per CU; where x's digits leave room for one only,
  // in workgroups of two.  A set meets at a barrier after every unit: with three rounds and more of
  // four times as many sets of 2 they are the faster (128256 x 4096: 40.9 us, sets of 8 45.0; but
  // 57344 x 8192, 1.75 rounds: 41.4 and 39.2, since a round's last units leave waves idle).
  const uint32_t cus = (uint32_t)std::max(rt->info.compute_units, 1);
  const uint32_t cap = a.mode == AMMON_GEMV_PLAIN_ARGMAX ? a.cand_cap : UINT32_MAX;
  const uint64_t a_cu = (uint64_t)p.row_blocks * cdiv(a.n, 128) / cus;
  int way = 2 * (lds_of(8) + 4096) > kLdsPerCu ? kW4Wide : p.row_blocks >= 3 * 8 * cus ? kW4Pairs : kW4Sets;
  auto grid_of = [&](int by) {
    if (by == kW4Flat) return std::min({p.row_blocks, cus, cap});
    return std::min({cdiv(p.row_blocks, by == kW4Wide ? 2 : by == kW4Pairs ? 4 : 1),
                     cus * (by == kW4Wide ? 1 : 2), cap});
  };
  const bool one = a.n <= 8 * 128 * AMMON_W4_CHUNK && grid_of(kW4One) == p.row_blocks;
  const bool flat = cdiv(p.row_blocks, grid_of(kW4Flat)) <= AMMON_W4_UNITS;
  if (way == kW4Sets && one) way = kW4One;
  if (p.row_blocks >= cus && a_cu >= 64 && a_cu <= 384 && flat) way = kW4Flat;
  if (rt->w4_way >= 0) {
    way = rt->w4_way;
    AMMON_CHECK((one || way != kW4One) && (flat || way != kW4Flat),
                "%s: the way chosen does not take this call", what);
  }
  uint32_t grid = grid_of(way);
  VALIDATE_ONLY();
  if (grid_out) *grid_out = grid;
  DeviceGuard guard(rt->device);
  void *args[] = {&p.w0, &p.x, &p.norm_w, &p.n, &p.norm_dtype, &p.row_blocks, &grid, &p.w1, &p.w2, &p};
  const hipError_t e =
      hipModuleLaunchKernel(rt->k.w4_gemv[way][a.mode], grid, 1, 1, way >= kW4Wide ? 1024 : 512, 1, 1,
                            (uint32_t)lds_of(way == kW4Pairs ? 2 : way == kW4Flat ? 1 : 8),
                            stream ? (hipStream_t)stream : rt->stream, args, nullptr);
  if (e != hipSuccess) return hip_error(e, what);
  return AMMON_OK;
}

}  // namespace ammon_rt

extern "C" {

ammon_status ammon_w4_choose(ammon_runtime *rt, const char *tile, const char *way) {
  REQUIRE_RT();
  int tiles[2] = {-1, -1}, ranges = 0, w = -1;
  if (tile) {
    const char *slash = std::strchr(tile, '/');
    const size_t len = slash ? (size_t)(slash - tile) : std::strlen(tile);
    auto called = [&](const char *name) { return std::strlen(name) == len && !std::strncmp(name, tile, len); };
    for (int q = 0; q < 2; ++q)
      for (tiles[q] = 0; tiles[q] < kW4Tiles && !called(kW4Tile[q][tiles[q]].name);) ++tiles[q];
    AMMON_CHECK(std::min(tiles[0], tiles[1]) < kW4Tiles, "w4_choose: no tile is called %.40s", tile);
    if (slash) {
      ranges = slash[1] - '0';
      AMMON_CHECK((ranges == 1 || ranges == 2 || ranges == 4 || ranges == 8) && !slash[2],
                  "w4_choose: %.40s: ranges are 1, 2, 4 or 8", tile);
    }
  }
  if (way) {
    for (w = 0; w < kW4Ways && std::strcmp(way, kW4WayName[w]);) ++w;
    AMMON_CHECK(w < kW4Ways, "w4_choose: no way is called %.40s", way);
  }
  rt->w4_tile[0] = tiles[0];
  rt->w4_tile[1] = tiles[1];
  rt->w4_ranges = (uint32_t)ranges;
  rt->w4_way = w;
  return AMMON_OK;
}

size_t ammon_w4_bytes(uint32_t d, uint32_t n) { return (size_t)cdiv(d, 16) * cdiv(n, 128) * 1056; }

ammon_status ammon_w4_store(ammon_runtime *rt, ammon_stream stream, const void *w, ammon_dtype w_dtype,
                            uint32_t d, uint32_t n, void *out) {
  REQUIRE_RT();
  AMMON_CHECK(w && out, "w4_store: NULL matrix or output");
  AMMON_CHECK(valid_dtype(w_dtype), "w4_store: unknown dtype %d", (int)w_dtype);
  TRY(shape_check("w4_store", d, n));
  TRY(aligned("w4_store", out, "W4 weights"));
  AMMON_CHECK(!overlaps(w, (size_t)d * n * dsize(w_dtype), out, ammon_w4_bytes(d, n)),
              "w4_store: the output overlaps the matrix");
  VALIDATE_ONLY();
  ammon_k_w4 p = {};
  p.w = w;
  p.w4 = out;
  p.d = d;
  p.n = n;
  p.dtype = (uint32_t)w_dtype;
  return launch(rt, stream, rt->k.w4_store, cdiv(d, 16), std::min(cdiv(n, 128), 65535u), 0, p, "w4_store");
}

ammon_status ammon_w4_load(ammon_runtime *rt, ammon_stream stream, const void *w4, uint32_t d, uint32_t n,
                           void *out, ammon_dtype out_dtype) {
  REQUIRE_RT();
  AMMON_CHECK(w4 && out, "w4_load: NULL weights or output");
  AMMON_CHECK(valid_dtype(out_dtype), "w4_load: unknown output dtype %d", (int)out_dtype);
  TRY(shape_check("w4_load", d, n));
  TRY(aligned("w4_load", w4, "W4 weights"));
  AMMON_CHECK(!overlaps(out, (size_t)d * n * dsize(out_dtype), w4, ammon_w4_bytes(d, n)),
              "w4_load: the output overlaps the weights");
  VALIDATE_ONLY();
  ammon_k_w4 p = {};
  p.w4 = (void *)w4;
  p.out = out;
  p.d = d;
  p.n = n;
  p.dtype = (uint32_t)out_dtype;
  return launch(rt, stream, rt->k.w4_load, cdiv(d, 16), std::min(cdiv(n, 128), 65535u), 0, p, "w4_load");
}

size_t ammon_q8_bytes(ammon_dtype dtype, uint32_t tokens, uint32_t n) {
  if (!valid_digits(dtype)) return 0;
  return (size_t)cdiv(tokens, 16) * cdiv(n, 128) * (2048 * (dtype == AMMON_Q8 ? 1 : 3) + 64);
}

ammon_status ammon_q8_store(ammon_runtime *rt, ammon_stream stream, const float *x, uint32_t tokens, uint32_t n,
                            void *out, ammon_dtype dtype) {
  REQUIRE_RT();
  return q8_rows(rt, stream, x, nullptr, nullptr, nullptr, AMMON_F32, 0.f, tokens, n, out, dtype, "q8_store");
}

ammon_status ammon_rmsnorm_q8(ammon_runtime *rt, ammon_stream stream, const float *x, const float *residual,
                              float *sum, const void *weight, ammon_dtype weight_dtype, float eps,
                              uint32_t tokens, uint32_t n, void *out, ammon_dtype dtype) {
  REQUIRE_RT();
  AMMON_CHECK(weight != nullptr, "rmsnorm_q8: parameter `weight` is NULL");
  AMMON_CHECK(valid_dtype(weight_dtype), "rmsnorm_q8: unknown weight dtype %d", (int)weight_dtype);
  AMMON_CHECK(std::isfinite(eps) && eps >= 0.f, "rmsnorm_q8: eps must be finite and >= 0");
  AMMON_CHECK(!residual == !sum, "rmsnorm_q8: residual and sum go together");
  return q8_rows(rt, stream, x, residual, sum, weight, weight_dtype, eps, tokens, n, out, dtype, "rmsnorm_q8");
}

ammon_status ammon_q8_load(ammon_runtime *rt, ammon_stream stream, const void *rows, ammon_dtype dtype,
                           uint32_t tokens, uint32_t n, float *out) {
  REQUIRE_RT();
  AMMON_CHECK(rows && out, "q8_load: NULL rows or output");
  AMMON_CHECK(valid_digits(dtype), "q8_load: rows are AMMON_Q8 or AMMON_Q24, not dtype %d", (int)dtype);
  TRY(shape_check("q8_load", tokens, n));
  TRY(aligned("q8_load", rows, "rows"));
  AMMON_CHECK(!overlaps(out, (size_t)tokens * n * 4, rows, ammon_q8_bytes(dtype, tokens, n)),
              "q8_load: the output overlaps the rows");
  VALIDATE_ONLY();
  ammon_k_q8 p = {};
  p.rows = (void *)rows;
  p.sum = out;
  p.tokens = tokens;
  p.n = n;
  p.vec = n % 4 == 0;
  const uint64_t waves = (uint64_t)cdiv(tokens, 16) * cdiv(n, 128);
  return launch(rt, stream, rt->k.q8_load[dtype == AMMON_Q24],
                (uint32_t)std::min<uint64_t>((waves + kWaves - 1) / kWaves, 1u << 20), 1, 0, p, "q8_load");
}

ammon_status ammon_prefill_gemm_w4(ammon_runtime *rt, ammon_stream stream, const void *w, uint32_t d, uint32_t n,
                                   const void *x, ammon_dtype x_dtype, uint32_t tokens, float *y,
                                   const float *residual, void *workspace, size_t workspace_bytes) {
  REQUIRE_RT();
  W4GemmArgs a = {};
  a.mode = residual ? AMMON_GEMV_RESIDUAL : AMMON_GEMV_PLAIN;
  a.w0 = w;
  a.d = d;
  a.n = n;
  a.rows = d;
  a.tokens = tokens;
  a.x = x;
  a.x_dtype = x_dtype;
  a.residual = residual;
  a.y = y;
  a.y_bytes = (size_t)tokens * d * 4;
  a.ws = workspace;
  a.ws_bytes = workspace ? workspace_bytes : 0;
  return w4_gemm(rt, stream, a, "prefill_gemm_w4");
}

ammon_status ammon_prefill_gate_up_swiglu_w4(ammon_runtime *rt, ammon_stream stream, const void *x,
                                             ammon_dtype x_dtype, uint32_t tokens, const void *w1,
                                             const void *w3, uint32_t dim, uint32_t hidden, float *hb) {
  REQUIRE_RT();
  AMMON_CHECK(w1 && w3, "prefill_gate_up_swiglu_w4: NULL w1 or w3");
  AMMON_CHECK((uint64_t)hidden * 2 < (1ull << 31), "prefill_gate_up_swiglu_w4: too many rows");
  W4GemmArgs a = {};
  a.mode = AMMON_GEMV_SWIGLU;
  a.w0 = w1;
  a.w1 = w3;
  a.d = hidden;
  a.n = dim;
  a.rows = 2 * hidden;
  a.tokens = tokens;
  a.x = x;
  a.x_dtype = x_dtype;
  a.y = hb;
  a.y_bytes = (size_t)tokens * hidden * 4;
  return w4_gemm(rt, stream, a, "prefill_gate_up_swiglu_w4");
}

ammon_status ammon_prefill_qkv_rope_w4(ammon_runtime *rt, ammon_stream stream, const void *x,
                                       ammon_dtype x_dtype, uint32_t tokens, const void *wq, const void *wk,
                                       const void *wv, uint32_t dim, uint32_t q_heads, uint32_t kv_heads,
                                       uint32_t head, float *q, float *k, float *v, uint32_t seq,
                                       const ammon_decode_step *step, const float *table, void *workspace,
                                       size_t workspace_bytes) {
  REQUIRE_RT();
  return w4_qkv(rt, stream, x, x_dtype, tokens, wq, wk, wv, dim, q_heads, kv_heads, head, q, k, v, AMMON_F32,
                true, seq, step, table, workspace, workspace_bytes, "prefill_qkv_rope_w4");
}

ammon_status ammon_prefill_qkv_rope_store_w4(ammon_runtime *rt, ammon_stream stream, const void *x,
                                             ammon_dtype x_dtype, uint32_t tokens, const void *wq,
                                             const void *wk, const void *wv, uint32_t dim, uint32_t q_heads,
                                             uint32_t kv_heads, uint32_t head, float *q, void *k_cache,
                                             void *v_cache, ammon_dtype kv_dtype, uint32_t seq,
                                             const ammon_decode_step *step, const float *table,
                                             void *workspace, size_t workspace_bytes) {
  REQUIRE_RT();
  return w4_qkv(rt, stream, x, x_dtype, tokens, wq, wk, wv, dim, q_heads, kv_heads, head, q, k_cache, v_cache,
                kv_dtype, false, seq, step, table, workspace, workspace_bytes, "prefill_qkv_rope_store_w4");
}

}  // extern "C"
