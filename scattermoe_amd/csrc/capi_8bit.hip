// extern "C" entry points of the products on 8-bit operands and of the passes around them: argument checks, the workspace's layout,
// the launches of a call.  Nothing here allocates; every launch goes to the caller's stream.
#include "eight_bit.hpp"

namespace smoe {

static bool float_type(int d) { return d == SMOE_F32 || d == SMOE_BF16 || d == SMOE_F16; }
static bool act_ok(int a) { return a == SMOE_ACT_SILU || a == SMOE_ACT_SILU_GATE_FIRST; }
static constexpr int64_t MOST = 0x3fffffff;                        // columns
static constexpr int64_t WIDEST = 1 << 21;                         // of a product: the rows of a tile are 32-bit offsets from its first

// pieces of a workspace, each at a multiple of 256 bytes
struct Carver {
  char* base;
  size_t used = 0;
  template <typename T = uint8_t>
  T* take(int64_t bytes) {
    T* p = base ? (T*)(base + used) : nullptr;
    used += ((size_t)bytes + 255) / 256 * 256;
    return p;
  }
};

// Rows of 8-bit activations of a product of L rows that come by token: the tokens once, or once per slot where those are scaled, and the product looks
// them up; a copy for each row, in the rows' order, where they pass the 32-bit offsets of a look-up.  All entry points ask here: the
// number of rows does not tell the ways apart (at one expert per token both have L).
struct SourceRows { bool looked_up; int64_t rows; };
static SourceRows source_rows(int64_t L, int64_t K, int fan, int x_grouped, bool scaled) {
  const int64_t held = scaled || x_grouped ? L : L / fan;
  const bool looked_up = !x_grouped && held * block_row(K) < (1LL << 32);
  return {looked_up, looked_up ? held : L};
}
static float* take_partial(Carver& c, int64_t floats) { return floats ? c.take<float>(floats * 4) : nullptr; }
struct Rows8Bit { uint8_t* q; uint8_t* s; int64_t rows; };
static Rows8Bit take_rows(Carver& c, int64_t rows, int64_t K) {
  Rows8Bit r{nullptr, nullptr, rows};
  r.q = c.take(rows * block_row(K) + QB);                          // (a product reads a slice further, and does not look at it)
  r.s = c.take(rows * scale_row(K));
  return r;
}
static int quantize(const Rows8Bit& r, const void* X, int64_t sxm, const int64_t* idx, int fan, const void* coeff, int64_t K, int dtype,
                    hipStream_t st, QuantRowsArgs::Clear clear = {}) {
  QuantRowsArgs a{X, sxm, idx, fan, coeff, coeff && !idx ? r.rows / fan : r.rows, K, r.q, r.s, r.rows, block_row(K), clear};
  return launch_quantize_rows(a, dtype, st);
}

// the rows (L, N) of `dtype` that a product writes, for zeros where the routing dropped some
static QuantRowsArgs::Clear dropped_rows(void* Y, int64_t sym, int64_t L, int64_t N, int dtype, const int64_t* off, int E) {
  const int64_t size = dtype == SMOE_F32 ? 4 : 2;
  return {(char*)Y, L, N * size, sym * size, off + E - 1};
}

static int weight_checks(const char* who, const smoe_weight_8bit* w, int64_t rows, int64_t cols) {
  if (!w || !w->q || !w->s) { set_error("%s: NULL weight", who); return SMOE_ERR_NULL; }
  if (((uintptr_t)w->q | w->q_expert) & 15) { set_error("%s: an expert's weights start at multiples of 16 bytes", who); return SMOE_ERR_SHAPE; }
  // (an expert's scales are 32-bit offsets from its first)
  if (w->s_row < 0 || w->s_col < 0 || scale_blocks(rows) * w->s_row + scale_blocks(cols) * w->s_col > (1LL << 28)) {
    set_error("%s: an expert's scales lie too far apart", who);
    return SMOE_ERR_RANGE;
  }
  return 0;
}
static Product8Args product(const Rows8Bit& x, const smoe_weight_8bit* w, bool transposed, const void* b, int64_t sbe, int64_t sbn, void* Y,
                            int64_t sym, const int64_t* idx, const int64_t* off, int64_t L, int64_t K, int64_t N, int E, int fan,
                            int x_grouped, int y_grouped) {
  Product8Args a{};
  a.X = x.q, a.XS = x.s;
  a.W = (const uint8_t*)w->q, a.swe = w->q_expert, a.swn = padded_row(K);
  a.WS = w->s, a.sse = w->s_expert, a.ssn = transposed ? w->s_col : w->s_row, a.ssk = transposed ? w->s_row : w->s_col;
  a.ws_f32 = w->s_float32;
  a.b = b, a.sbe = sbe, a.sbn = sbn;
  a.Y = Y, a.sym = sym;
  a.idx = idx, a.off = off;
  a.L = (int)L, a.K = (int)padded_row(K), a.N = (int)N, a.E = E, a.fan = fan, a.x_grouped = x_grouped, a.y_grouped = y_grouped;
  return a;
}

static Few8Args few(const smoe_weight_8bit* w, const void* b, int64_t sbe, int64_t sbn, void* Y, int64_t sym, int out_dtype, const int64_t* ids,
                    const int64_t* idx, const int64_t* off, int64_t L, int64_t K, int64_t N, int E, int fan, int x_grouped, int y_grouped, int act) {
  Few8Args a{};
  a.W = (const uint8_t*)w->q, a.swe = w->q_expert;
  a.WS = w->s, a.sse = w->s_expert, a.ssn = w->s_row, a.ssk = w->s_col, a.ws_f32 = w->s_float32;
  a.b = b, a.sbe = sbe, a.sbn = sbn;
  a.Y = Y, a.sym = sym, a.out_dtype = out_dtype;
  a.ids = ids, a.idx = idx, a.off = off;
  a.L = (int)L, a.K = (int)K, a.N = (int)N, a.E = E, a.fan = fan, a.x_grouped = x_grouped, a.y_grouped = y_grouped, a.act = act;
  return a;
}
// Streams over the weights instead of tiles, for products that contract K values (the shortest of a layer).  Layers, us at 2, 4, 6, 8, 11 rows per
// expert, even loads: 8 experts, 4096 / 14336 249, 255, 260, 265, 268, in tiles of 64 rows 331 from 11 on; 32 experts, 2880 / 2880 -, 180, 196, 199, -,
// tiles 186, 190, 190; 128 experts, 2048 / 768 127, 141, 158, 166, -, tiles 132, 141, 145, 145.  Products: 16 experts, 4096 -> 14336 at 10, 12, 15 rows
// 158, 169, 181, tiles 184 and more.  (32768 rows: a segment per expert or 8 rows is a grid's second side.)
static bool few_rows_pay(int64_t L, int64_t K, int E) { return L <= (K >= 4096 ? 12 : 4) * (int64_t)E && L <= 32768; }

// Products of a layer that multiply exactly (SCALES_EXACT), beside those of float32 rows: of float16 rows the ones whose results go to 8 bits again.  A
// hidden value, or a gradient, whose sum is 1e-5 off may fall to the other side of a border between two 8-bit values, a step of 2^-4,
// and such steps cost 1e-3 of the result, five times float16's own rounding (65 tokens to 4 of 32 experts, 2880 / 2880, against 64 bits:
// 1.4e-3, so 2.1e-4, as the plain form).  Bfloat16 rounds to 1.7e-3 by itself, which the steps make 2.0e-3 to 2.2e-3.
static bool product_exact(int dtype) { return dtype == SMOE_F32; }
static bool inner_exact(int dtype) { return dtype != SMOE_BF16; }

}  // namespace smoe

using namespace smoe;

extern "C" {

int64_t smoe_row_8bit_bytes(int64_t K) { return padded_row(K); }
int64_t smoe_row_8bit_scales(int64_t K) { return scale_row(K); }

int smoe_quantize_rows(const void* X, int64_t sxm, int64_t rows, int64_t K, void* Q, void* S, int dtype, void* stream) {
  set_error("%s", "");
  if (!float_type(dtype)) { set_error("smoe_quantize_rows: unknown dtype %d", dtype); return SMOE_ERR_DTYPE; }
  if (rows < 0 || K < 0) { set_error("smoe_quantize_rows: bad sizes"); return SMOE_ERR_SHAPE; }
  if (K > MOST) { set_error("smoe_quantize_rows: size beyond int32"); return SMOE_ERR_RANGE; }
  if (rows == 0 || K == 0) return 0;
  if (!X || !Q || !S) { set_error("smoe_quantize_rows: NULL pointer"); return SMOE_ERR_NULL; }
  if ((uintptr_t)Q & 15) { set_error("smoe_quantize_rows: rows in 8 bits start at multiples of 16 bytes"); return SMOE_ERR_SHAPE; }
  QuantRowsArgs a{X, sxm, nullptr, 1, nullptr, rows, K, (uint8_t*)Q, (uint8_t*)S, rows, padded_row(K), {}};
  return launch_quantize_rows(a, dtype, (hipStream_t)stream);
}

int smoe_quantize_weights(const void* W, int64_t swe, int64_t swn, int E, int64_t N, int64_t K, void* Q, void* QT, void* S, int dtype,
                          void* stream) {
  set_error("%s", "");
  if (!float_type(dtype)) { set_error("smoe_quantize_weights: unknown dtype %d", dtype); return SMOE_ERR_DTYPE; }
  if (E < 0 || N < 0 || K < 0) { set_error("smoe_quantize_weights: bad sizes"); return SMOE_ERR_SHAPE; }
  if (K > MOST || N > MOST) { set_error("smoe_quantize_weights: size beyond int32"); return SMOE_ERR_RANGE; }
  if (E == 0 || N == 0 || K == 0) return 0;
  if (!W || !Q || !S) { set_error("smoe_quantize_weights: NULL pointer"); return SMOE_ERR_NULL; }
  if (((uintptr_t)Q | (uintptr_t)QT) & 15) { set_error("smoe_quantize_weights: rows in 8 bits start at multiples of 16 bytes"); return SMOE_ERR_SHAPE; }
  QuantWeightsArgs a{W, swe, swn, E, N, K, (uint8_t*)Q, (uint8_t*)QT, (uint8_t*)S};
  return launch_quantize_weights(a, dtype, (hipStream_t)stream);
}

int smoe_dequantize_8bit(const void* Q, int64_t sqe, int64_t sqn, const void* S, int64_t sse, int64_t ssn, int64_t ssk, int scales_float32,
                         int block_rows, int E, int64_t N, int64_t K, void* Y, int dtype, void* stream) {
  set_error("%s", "");
  if (!float_type(dtype)) { set_error("smoe_dequantize_8bit: unknown dtype %d", dtype); return SMOE_ERR_DTYPE; }
  if (E < 0 || N < 0 || K < 0 || (block_rows != 1 && block_rows != QB)) { set_error("smoe_dequantize_8bit: bad sizes"); return SMOE_ERR_SHAPE; }
  if (K > MOST) { set_error("smoe_dequantize_8bit: size beyond int32"); return SMOE_ERR_RANGE; }
  if (E == 0 || N == 0 || K == 0) return 0;
  if (!Q || !S || !Y) { set_error("smoe_dequantize_8bit: NULL pointer"); return SMOE_ERR_NULL; }
  DequantArgs a{(const uint8_t*)Q, sqe, sqn, S, sse, ssn, ssk, scales_float32, block_rows, E, N, K, Y};
  return launch_dequantize(a, dtype, (hipStream_t)stream);
}

static int unit_checks(const char* who, int64_t rows, int64_t F, int act, int dtype) {
  if (!float_type(dtype)) { set_error("%s: unknown dtype %d", who, dtype); return SMOE_ERR_DTYPE; }
  if (rows < 0 || F < 0) { set_error("%s: bad sizes", who); return SMOE_ERR_SHAPE; }
  if (!act_ok(act)) { set_error("%s: unknown activation %d", who, act); return SMOE_ERR_SHAPE; }
  if (F > MOST) { set_error("%s: size beyond int32", who); return SMOE_ERR_RANGE; }
  return 0;
}

int smoe_glu_8bit_fwd(const void* pre, int64_t spm, void* h, void* P8, void* PS, int64_t rows, int64_t F, int act, int dtype, void* stream) {
  set_error("%s", "");
  if (int rc = unit_checks("smoe_glu_8bit_fwd", rows, F, act, dtype)) return rc;
  if (rows == 0 || F == 0) return 0;
  if (!pre || !h || !P8 || !PS) { set_error("smoe_glu_8bit_fwd: NULL pointer"); return SMOE_ERR_NULL; }
  if ((uintptr_t)P8 & 15) { set_error("smoe_glu_8bit_fwd: rows in 8 bits start at multiples of 16 bytes"); return SMOE_ERR_SHAPE; }
  UnitArgs a{pre, spm, h, nullptr, nullptr, (uint8_t*)P8, (uint8_t*)PS, rows, F, act};
  return launch_unit_fwd(a, dtype, (hipStream_t)stream);
}

int smoe_glu_8bit_bwd(const void* P8, const void* PS, const void* dh, int64_t sdh, void* dpre, void* h, int64_t rows, int64_t F, int act,
                      int dtype, void* stream) {
  set_error("%s", "");
  if (int rc = unit_checks("smoe_glu_8bit_bwd", rows, F, act, dtype)) return rc;
  if (rows == 0 || F == 0) return 0;
  if (!P8 || !PS || !dh || !dpre) { set_error("smoe_glu_8bit_bwd: NULL pointer"); return SMOE_ERR_NULL; }
  if ((uintptr_t)P8 & 15) { set_error("smoe_glu_8bit_bwd: rows in 8 bits start at multiples of 16 bytes"); return SMOE_ERR_SHAPE; }
  UnitBackArgs a{(const uint8_t*)P8, (const uint8_t*)PS, dh, sdh, dpre, nullptr, nullptr, h, rows, F, act};
  return launch_unit_bwd(a, dtype, (hipStream_t)stream);
}

static int product_checks(const char* who, int64_t L, int64_t K, int64_t N, int E, int fan, int dtype) {
  if (!float_type(dtype)) { set_error("%s: unknown dtype %d", who, dtype); return SMOE_ERR_DTYPE; }
  if (L < 0 || K <= 0 || N < 0 || E <= 0 || fan <= 0 || L % fan != 0) { set_error("%s: bad sizes", who); return SMOE_ERR_SHAPE; }
  if (L > 0x7fffffffLL || K > WIDEST || N > WIDEST) { set_error("%s: size beyond int32", who); return SMOE_ERR_RANGE; }
  return 0;
}
static int workspace_check(const char* who, size_t need, const void* workspace, size_t bytes) {
  if (workspace && bytes >= need && ((uintptr_t)workspace & 255) == 0) return 0;
  set_error("%s: a workspace of %zu bytes, 256-byte aligned, is needed, %zu given", who, need, workspace ? bytes : (size_t)0);
  return SMOE_ERR_WORKSPACE;
}

size_t smoe_linear_8bit_workspace_bytes(int64_t L, int64_t K, int64_t N, int E, int fan_out, int x_grouped, int scaled, int dtype) {
  if (L <= 0 || K <= 0 || N <= 0 || E <= 0 || fan_out <= 0) return 0;
  Carver c{nullptr};
  take_rows(c, source_rows(L, K, fan_out, x_grouped, scaled != 0).rows, K);
  if (!few_rows_pay(L, K, E)) c.take(product_8bit_floats(L, K, N, E, product_exact(dtype & ~SMOE_8BIT_Y_FLOAT32)) * 4);
  return c.used;
}

int smoe_linear_8bit(const void* X, int64_t sxm, const void* coeff, const smoe_weight_8bit* W, int transposed, const void* b, int64_t sbe,
                     int64_t sbn, void* Y, int64_t sym, const int64_t* idx, const int64_t* off, int64_t L, int64_t K, int64_t N, int E,
                     int fan_out, int x_grouped, int y_grouped, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  set_error("%s", "");
  const int out_dtype = dtype & SMOE_8BIT_Y_FLOAT32 ? SMOE_F32 : dtype;
  dtype &= ~SMOE_8BIT_Y_FLOAT32;
  if (int rc = product_checks("smoe_linear_8bit", L, K, N, E, fan_out, dtype)) return rc;
  if (L == 0 || N == 0) return 0;
  if (!X || !Y || !idx || !off) { set_error("smoe_linear_8bit: NULL pointer"); return SMOE_ERR_NULL; }
  if (coeff && x_grouped) { set_error("smoe_linear_8bit: rows that are scaled come by token"); return SMOE_ERR_SHAPE; }
  if (int rc = weight_checks("smoe_linear_8bit", W, transposed ? K : N, transposed ? N : K)) return rc;
  if (int rc = workspace_check("smoe_linear_8bit", smoe_linear_8bit_workspace_bytes(L, K, N, E, fan_out, x_grouped, coeff != nullptr, dtype), workspace, workspace_bytes)) return rc;
  Carver c{(char*)workspace};
  const SourceRows from = source_rows(L, K, fan_out, x_grouped, coeff != nullptr);
  const bool by_token = from.looked_up;
  const Rows8Bit x = take_rows(c, from.rows, K);
  const int fan = coeff ? 1 : fan_out;                             // rows of x per row of the product's left side
  const bool copies = !x_grouped && !by_token;
  if (int rc = quantize(x, X, sxm, copies ? idx : nullptr, fan_out, coeff, K, dtype, (hipStream_t)stream,
                        dropped_rows(Y, sym, L, N, out_dtype, off, E))) return rc;
  if (few_rows_pay(L, K, E)) {
    Few8Args a = few(W, b, sbe, sbn, Y, sym, out_dtype, nullptr, idx, off, L, K, N, E, fan, !by_token, y_grouped, 0);
    if (transposed) a.ssn = W->s_col, a.ssk = W->s_row;
    a.X = x.q, a.sxm = block_row(K), a.XS = x.s;
    return launch_few_rows_8bit(a, -1, dtype, EPI_ROWS, (hipStream_t)stream);
  }
  Product8Args a = product(x, W, transposed != 0, b, sbe, sbn, Y, sym, idx, off, L, K, N, E, fan, !by_token, y_grouped);
  a.partial = take_partial(c, product_8bit_floats(L, K, N, E, product_exact(dtype)));
  return launch_product_8bit(a, product_exact(dtype), dtype, out_dtype, (hipStream_t)stream);
}

int smoe_combine_f32(const void* Y, int64_t sym, const void* gates, int64_t sgt, int64_t sgk, const int64_t* experts, int E, void* out, int64_t som,
                     int64_t T, int k, int64_t N, int dtype, void* stream) {
  set_error("%s", "");
  if (!float_type(dtype)) { set_error("smoe_combine_f32: unknown dtype %d", dtype); return SMOE_ERR_DTYPE; }
  if (T < 0 || k <= 0 || N < 0 || (experts && E <= 0)) { set_error("smoe_combine_f32: bad sizes"); return SMOE_ERR_SHAPE; }
  if (T > 0x7fffffffLL || N > MOST) { set_error("smoe_combine_f32: size beyond int32"); return SMOE_ERR_RANGE; }
  if (T == 0 || N == 0) return 0;
  if (!Y || !out) { set_error("smoe_combine_f32: NULL pointer"); return SMOE_ERR_NULL; }
  return launch_slots_combine((const float*)Y, sym, gates, sgt, sgk, experts, E, out, som, T, k, (int)N, dtype, (hipStream_t)stream);
}

int smoe_gate_grad_f32(const void* Y, int64_t sym, const void* dOut, int64_t sdm, void* dgates, int64_t sgt, int64_t sgk, int64_t T, int k, int64_t N,
                       int dtype, void* stream) {
  set_error("%s", "");
  if (!float_type(dtype)) { set_error("smoe_gate_grad_f32: unknown dtype %d", dtype); return SMOE_ERR_DTYPE; }
  if (T < 0 || k <= 0 || N < 0) { set_error("smoe_gate_grad_f32: bad sizes"); return SMOE_ERR_SHAPE; }
  if (T > 0x7fffffffLL || T * k > 0x7fffffffLL || N > MOST) { set_error("smoe_gate_grad_f32: size beyond int32"); return SMOE_ERR_RANGE; }
  if (T == 0) return 0;
  if (!dgates || (N > 0 && (!Y || !dOut))) { set_error("smoe_gate_grad_f32: NULL pointer"); return SMOE_ERR_NULL; }
  return launch_slots_gate_grad((const float*)Y, sym, dOut, sdm, dgates, sgt, sgk, T, k, (int)N, dtype, (hipStream_t)stream);
}

// Streams multiply exactly anyhow, and pay against such tiles up to 16 rows per expert, the most that one reading of the weights takes.  Layers in float32,
// us at 8, 12, 16, 24 rows per expert, streams and tiles: 8 experts, 4096 / 14336 261, 268, 278, 414 and 515 from 8 on; 32 experts, 2880 / 2880
// 195, 204, 211, 316 and 325; 128 experts, 2048 / 768 162, 173, 179, 264 and 250.  In float16 the same streams, tiles 463, 276 and 219.
static bool streams_pay(int64_t L, int64_t d, int64_t F, int E, int dtype) {
  return few_rows_pay(L, d < F ? d : F, E) || (inner_exact(dtype) && L <= 16 * (int64_t)E && L <= 32768);
}

// How a layer goes.  Without an order of its rows: by their ids, two streams over the weights of the experts that they name.  Few rows per
// expert: streams over the weights, rows by expert.  Else tiles, with the unit behind the first product where it rides.
enum LayerWay { LAYER_BY_IDS, LAYER_FEW, LAYER_TILES, LAYER_TILES_UNIT };
static LayerWay layer_way(int64_t L, int64_t d, int64_t F, int E, bool ordered, bool keep, int dtype) {
  if (!ordered) return LAYER_BY_IDS;
  if (!keep && streams_pay(L, d, F, E, dtype)) return LAYER_FEW;
  return unit_rides(d, F) ? LAYER_TILES_UNIT : LAYER_TILES;
}
// the pieces of a gated layer's workspace
struct LayerPieces { Rows8Bit x, h; bool by_token; float* pre; float* hidden; float* rows; float* partial1; float* partial2; };
static LayerPieces layer_pieces(Carver& c, LayerWay way, int64_t L, int k, int64_t d, int64_t F, int E, int dtype) {
  LayerPieces p{};
  if (way == LAYER_BY_IDS) {
    p.hidden = c.take<float>(L * F * 4);
    p.rows = c.take<float>(L * d * 4);
    return p;
  }
  const SourceRows from = source_rows(L, d, k, 0, false);
  p.by_token = from.looked_up;
  p.x = take_rows(c, from.rows, d);
  p.h = take_rows(c, L, F);
  if (way == LAYER_FEW) p.hidden = c.take<float>(L * F * 4);
  if (way == LAYER_TILES) p.pre = c.take<float>(L * 2 * F * 4);
  if (way != LAYER_FEW) {                                          // (one after the other: the same piece for both products)
    const int64_t one = product_8bit_floats(L, d, 2 * F, E, inner_exact(dtype)), two = product_8bit_floats(L, F, d, E, product_exact(dtype));
    float* both = take_partial(c, one > two ? one : two);
    p.partial1 = one ? both : nullptr, p.partial2 = two ? both : nullptr;
  }
  return p;
}
size_t smoe_glu_mlp_8bit_workspace_bytes(int64_t T, int k, int64_t d, int64_t F, int E, int ordered, int keep, int dtype) {
  if (T <= 0 || k <= 0 || d <= 0 || F <= 0 || E <= 0) return 0;
  Carver c{nullptr};
  layer_pieces(c, layer_way(T * k, d, F, E, ordered != 0, keep != 0, dtype), T * k, k, d, F, E, dtype);
  return c.used;
}

int smoe_glu_mlp_8bit(const void* X, int64_t sxm, const void* gates, const int64_t* experts, const smoe_weight_8bit* W1, const void* b1,
                      int64_t sb1e, int64_t sb1n, const smoe_weight_8bit* W2, const void* b2, int64_t sb2e, int64_t sb2n, void* Y, void* OUT,
                      void* P8, void* PS, const int64_t* idx, const int64_t* off, int64_t T, int k, int64_t d, int64_t F, int E, int act,
                      int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  set_error("%s", "");
  hipStream_t st = (hipStream_t)stream;
  if (k <= 0 || F <= 0) { set_error("smoe_glu_mlp_8bit: bad sizes"); return SMOE_ERR_SHAPE; }
  if (int rc = product_checks("smoe_glu_mlp_8bit", T * k, d, F, E, k, dtype)) return rc;
  if (!act_ok(act)) { set_error("smoe_glu_mlp_8bit: unknown activation %d", act); return SMOE_ERR_SHAPE; }
  if (T == 0) return 0;
  const int64_t L = T * k;
  const bool ordered = idx != nullptr;
  const LayerWay way = layer_way(L, d, F, E, ordered, P8 != nullptr, dtype);
  if (!ordered && (L > SMOE_8BIT_FEW_ROWS || P8)) { set_error("smoe_glu_mlp_8bit: an order is needed for more than %d rows, and to keep P8", SMOE_8BIT_FEW_ROWS); return SMOE_ERR_NULL; }
  if (!X || !gates || !OUT || (P8 && !PS) || (ordered ? !Y || !off : !experts)) { set_error("smoe_glu_mlp_8bit: NULL pointer"); return SMOE_ERR_NULL; }
  if ((uintptr_t)P8 & 15) { set_error("smoe_glu_mlp_8bit: P8 starts at a multiple of 16 bytes"); return SMOE_ERR_SHAPE; }
  if (int rc = weight_checks("smoe_glu_mlp_8bit", W1, 2 * F, d)) return rc;
  if (int rc = weight_checks("smoe_glu_mlp_8bit", W2, d, F)) return rc;
  if (int rc = workspace_check("smoe_glu_mlp_8bit", smoe_glu_mlp_8bit_workspace_bytes(T, k, d, F, E, ordered, P8 != nullptr, dtype), workspace, workspace_bytes)) return rc;
  Carver c{(char*)workspace};
  const LayerPieces p = layer_pieces(c, way, L, k, d, F, E, dtype);
  if (way == LAYER_BY_IDS) {
    Few8Args a = few(W1, b1, sb1e, sb1n, p.hidden, F, SMOE_F32, experts, nullptr, nullptr, L, d, 2 * F, E, k, 0, 1, act);
    a.X = X, a.sxm = sxm, a.x_vec = ((uintptr_t)X & 15) == 0 && sxm * (dtype == SMOE_F32 ? 4 : 2) % 16 == 0;
    if (int rc = launch_few_rows_8bit(a, dtype, dtype, EPI_UNIT, st)) return rc;
    a = few(W2, b2, sb2e, sb2n, p.rows, d, SMOE_F32, experts, nullptr, nullptr, L, F, d, E, 1, 1, 1, act);
    a.X = p.hidden, a.sxm = F, a.x_vec = F % 4 == 0;
    if (int rc = launch_few_rows_8bit(a, SMOE_F32, dtype, EPI_ROWS, st)) return rc;
    return launch_few_combine(p.rows, gates, experts, OUT, (int)T, k, (int)d, E, dtype, st);
  }
  const bool by_token = p.by_token;
  if (int rc = quantize(p.x, X, sxm, by_token ? nullptr : idx, k, nullptr, d, dtype, st, dropped_rows(Y, d, L, d, SMOE_F32, off, E))) return rc;
  if (way == LAYER_FEW) {
    Few8Args a = few(W1, b1, sb1e, sb1n, p.hidden, F, SMOE_F32, nullptr, idx, off, L, d, 2 * F, E, k, !by_token, 1, act);
    a.X = p.x.q, a.sxm = block_row(d), a.XS = p.x.s;
    if (int rc = launch_few_rows_8bit(a, -1, dtype, EPI_UNIT, st)) return rc;
    if (int rc = quantize(p.h, p.hidden, F, nullptr, 1, nullptr, F, SMOE_F32, st)) return rc;
    a = few(W2, b2, sb2e, sb2n, Y, d, SMOE_F32, nullptr, idx, off, L, F, d, E, 1, 1, 0, act);
    a.X = p.h.q, a.sxm = block_row(F), a.XS = p.h.s;
    if (int rc = launch_few_rows_8bit(a, -1, dtype, EPI_ROWS, st)) return rc;
    return launch_slots_combine((const float*)Y, d, gates, k, 1, experts, E, OUT, d, T, k, (int)d, dtype, st);
  }
  Product8Args a = product(p.x, W1, false, b1, sb1e, sb1n, p.pre, 2 * F, idx, off, L, d, 2 * F, E, k, !by_token, 1);
  a.partial = p.partial1;
  if (way == LAYER_TILES_UNIT) {
    a.H8 = p.h.q, a.HS = p.h.s, a.P8 = (uint8_t*)P8, a.PS = (uint8_t*)PS, a.act = act;
    if (int rc = launch_product_8bit(a, inner_exact(dtype), dtype, SMOE_F32, st, EPI_UNIT)) return rc;
  } else {
    if (int rc = launch_product_8bit(a, inner_exact(dtype), dtype, SMOE_F32, st)) return rc;
    UnitArgs u{p.pre, 2 * F, nullptr, p.h.q, p.h.s, (uint8_t*)P8, (uint8_t*)PS, L, F, act};
    if (int rc = launch_unit_fwd(u, SMOE_F32, st)) return rc;
  }
  a = product(p.h, W2, false, b2, sb2e, sb2n, Y, d, idx, off, L, F, d, E, 1, 1, 0);
  a.partial = p.partial2;
  if (int rc = launch_product_8bit(a, product_exact(dtype), dtype, SMOE_F32, st)) return rc;
  return launch_slots_combine((const float*)Y, d, gates, k, 1, experts, E, OUT, d, T, k, (int)d, dtype, st);
}

struct BackPieces { Rows8Bit dy, dp; bool by_slot; float* dh; float* partial1; float* partial2; };
static BackPieces back_pieces(Carver& c, int64_t L, int k, int64_t d, int64_t F, int E, int dtype) {
  BackPieces p{};
  const SourceRows from = source_rows(L, d, k, 0, true);
  p.by_slot = from.looked_up;
  p.dy = take_rows(c, from.rows, d);
  p.dp = take_rows(c, L, 2 * F);
  p.dh = unit_grad_rides(F) ? nullptr : c.take<float>(L * F * 4);
  const int64_t one = product_8bit_floats(L, d, F, E, inner_exact(dtype)), two = product_8bit_floats(L, 2 * F, d, E, product_exact(dtype));
  float* both = take_partial(c, one > two ? one : two);
  p.partial1 = one ? both : nullptr, p.partial2 = two ? both : nullptr;
  return p;
}
size_t smoe_glu_mlp_8bit_bwd_workspace_bytes(int64_t T, int k, int64_t d, int64_t F, int E, int dtype) {
  if (T <= 0 || k <= 0 || d <= 0 || F <= 0 || E <= 0) return 0;
  Carver c{nullptr};
  back_pieces(c, T * k, k, d, F, E, dtype);
  return c.used;
}

int smoe_glu_mlp_8bit_bwd(const void* DOUT, int64_t sdm, const void* gates, const smoe_weight_8bit* W1T, const smoe_weight_8bit* W2T,
                          const void* P8, const void* PS, void* DROWS, void* DX, const int64_t* idx, const int64_t* off, int64_t T, int k,
                          int64_t d, int64_t F, int E, int act, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  set_error("%s", "");
  hipStream_t st = (hipStream_t)stream;
  if (k <= 0 || F <= 0) { set_error("smoe_glu_mlp_8bit_bwd: bad sizes"); return SMOE_ERR_SHAPE; }
  if (int rc = product_checks("smoe_glu_mlp_8bit_bwd", T * k, F, d, E, k, dtype)) return rc;
  if (!act_ok(act)) { set_error("smoe_glu_mlp_8bit_bwd: unknown activation %d", act); return SMOE_ERR_SHAPE; }
  if (T == 0 || d == 0) return 0;
  if (!DOUT || !gates || !P8 || !PS || !DROWS || !DX || !idx || !off) { set_error("smoe_glu_mlp_8bit_bwd: NULL pointer"); return SMOE_ERR_NULL; }
  if ((uintptr_t)P8 & 15) { set_error("smoe_glu_mlp_8bit_bwd: P8 starts at a multiple of 16 bytes"); return SMOE_ERR_SHAPE; }
  if (int rc = weight_checks("smoe_glu_mlp_8bit_bwd", W1T, 2 * F, d)) return rc;
  if (int rc = weight_checks("smoe_glu_mlp_8bit_bwd", W2T, d, F)) return rc;
  if (int rc = workspace_check("smoe_glu_mlp_8bit_bwd", smoe_glu_mlp_8bit_bwd_workspace_bytes(T, k, d, F, E, dtype), workspace, workspace_bytes)) return rc;
  const int64_t L = T * k;
  Carver c{(char*)workspace};
  const BackPieces p = back_pieces(c, L, k, d, F, E, dtype);
  const bool by_slot = p.by_slot;
  if (int rc = quantize(p.dy, DOUT, sdm, by_slot ? nullptr : idx, k, gates, d, dtype, st, dropped_rows(DROWS, d, L, d, SMOE_F32, off, E))) return rc;
  Product8Args a = product(p.dy, W2T, true, nullptr, 0, 0, p.dh, F, idx, off, L, d, F, E, 1, !by_slot, 1);
  a.partial = p.partial1;
  if (!p.dh) {
    a.H8 = p.dp.q, a.HS = p.dp.s, a.P8 = (uint8_t*)P8, a.PS = (uint8_t*)PS, a.act = act;
    if (int rc = launch_product_8bit(a, inner_exact(dtype), dtype, SMOE_F32, st, EPI_UNIT_GRAD)) return rc;
  } else {
    if (int rc = launch_product_8bit(a, inner_exact(dtype), dtype, SMOE_F32, st)) return rc;
    UnitBackArgs u{(const uint8_t*)P8, (const uint8_t*)PS, p.dh, F, nullptr, p.dp.q, p.dp.s, nullptr, L, F, act};
    if (int rc = launch_unit_bwd(u, SMOE_F32, st)) return rc;
  }
  a = product(p.dp, W1T, true, nullptr, 0, 0, DROWS, d, idx, off, L, 2 * F, d, E, 1, 1, 0);
  a.partial = p.partial2;
  if (int rc = launch_product_8bit(a, product_exact(dtype), dtype, SMOE_F32, st)) return rc;
  return launch_slots_combine((const float*)DROWS, d, nullptr, 0, 0, nullptr, E, DX, d, T, k, (int)d, dtype, st);
}

}  // extern "C"
