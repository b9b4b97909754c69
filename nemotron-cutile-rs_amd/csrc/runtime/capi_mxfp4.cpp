// Device entry points of the MXFP4 operators: validate on the host, then enqueue.
#include <algorithm>
#include <cstdint>

#include "../kernels/mx_numerics.h"
#include "nh_runtime.h"

using namespace nh;

namespace {

// Rows that one launch takes straight from x: what the kernel quantizes, an
// MFMA operand of 16 rows, and holds, eight waves of 16 K tiles.
constexpr size_t kMxRowsMax = 16;
constexpr size_t kMxRowsMaxK = 16384;

// Rows of codes that stream the weights, and the others go to the GEMM.  The
// streaming form holds K to 8192, 32 rows a pass past 4096 and 64 below, and
// reads the weights once a pass; the GEMM's time is a chain of stages along K
// while it has few tiles.  us, streamed / GEMM, each with its quantization
// (192 products of 17..64 rows, K 512..8192, 256..32768 columns: the choice is
// within 9% of the better one; streaming them all took up to 1.8 times as long):
//   64 rows -> 4096:  K 1024 11.1 / 7.6, 2048 12.6 / 9.5, 2688 10.0 / 11.4, 4096 12.8 / 13.2, 8192 20.1 / 20.9
//   64 rows -> 16384: K 2688 14.1 / 12.7, 4096 18.1 / 15.4, 8192 34.3 / 24.6
//   32 rows -> 8192:  K 1024 9.5 / 8.2, 2048 10.3 / 10.1, 4096 11.2 / 14.0, 8192 15.8 / 22.2
//   128 rows -> 4096: K 4096 20.4 / 13.3
bool mx_streams(size_t m, size_t n, size_t k) {
    return m <= 64 && k > 2048 && k <= 8192 && (m <= 32 || n * (k <= 4096 ? 1 : 2) <= 8192);
}

// K tiles that each of a group's waves owns (at most eight waves): 2, 4, 8, 16
// (index 0..3).  More per wave where K leaves a wave too few loads to hide
// their latency, and the other waves go to groups of their own.  32, 64 and 128
// K tiles are what eight waves of 4, 8 and 16 hold (fewer waves of more are
// slower: 4096 -> 16384 at m = 1 10.7 us by fours, 11.5 by eights); 8 is where
// twos and fours cross (1 x 1024 -> 4096 6.2 and 6.5, -> 16384 7.2 and 7.0; 2048
// -> 16384 8.6 and 7.8).
int mx_split(int kt) { return kt <= 8 ? 0 : kt <= 32 ? 1 : kt <= 64 ? 2 : 3; }

// A launch holds fewer than 2^32 threads in a dimension.
bool launchable(uint64_t workgroups, uint64_t threads) { return workgroups * threads < (1ull << 32); }

// A row of `cols` values in `rows`: what the conversions address.
nh_status check_mx_rows(size_t rows, size_t cols, nh_error* err) {
    size_t t;
    if (!mul_ok(rows, cols, &t) || t >= (1ull << 48)) return set_error(err, NH_INVALID_SHAPE, "rows * cols overflows");
    // a workgroup of 256 takes 1024 groups of eight values (so indices stay within the 38 bits of a non-finite word)
    if (rows > (size_t)kMaxGrid || cols > (size_t)kMaxGrid - 64 ||
        !launchable((rows * mx_row_blocks(cols) * 4 + 1023) / 1024, 256))
        return set_error(err, NH_UNSUPPORTED, "rows and cols must be < 2^31 and rows * ceil(cols / 32) <= 2^32 - 256");
    return NH_OK;
}

unsigned mx_unit_grid(int64_t units) { return (unsigned)((units + 1023) / 1024); }

// Rows that one pass of the few-row product takes (codes): as few as hold them
// all (17 x 4096 -> 16384: 19.6 us in passes of 16, 13.9 of 32, 14.9 of 64; 40
// rows 26.1, 21.9, 16.4).
int mx_pass_rows(size_t rows, int kt) { return rows <= 16 ? 16 : rows <= 32 || mx_split(kt) == 2 ? 32 : 64; }

// The few-row product: fills the launch shape into `a` and launches kernel
// first + split (16 rows at a time), or with as many rows, which are codes, the
// forms of 32 and 64 that follow it (K past 4096 has none of 64).
nh_status launch_mx_stream(nh_context* ctx, KernelId first, MxStreamArgs a, size_t rows, bool requant,
                           unsigned workgroups, unsigned experts, nh_stream stream, nh_error* err) {
    const int split = mx_split(a.kt), c = 2 << split, t = requant ? 2 : 1;
    const int pass = mx_pass_rows(rows, a.kt), form = pass == 16 ? 0 : pass == 32 ? 1 : 2;
    a.row_blocks = 1 << form;
    a.waves = (a.kt + c - 1) / c;
    a.groups = 8 / a.waves;
    // h's units cover its whole K tiles: their blocks past N are written as zeros
    const unsigned units = requant ? 4 * (unsigned)mx_k_tiles((uint64_t)a.N) : (unsigned)((a.N + 15) / 16);
    // a run's bias lies in LDS: at most 16 KiB
    const unsigned least = (units + 255 / t) / (256 / t);
    const unsigned gx = std::max(1u, std::min(units, std::max(workgroups, least)));
    a.run = (int)(units / gx);
    a.longer = (int)(units % gx);
    const size_t lds = (size_t)2 * t * a.row_blocks * a.waves * a.groups * 1024 + (a.bias ? (size_t)(a.run + 1) * t * 16 * 4 : 0);
    return launch(ctx, (KernelId)(first + 3 * form + split), gx, 64u * a.waves * a.groups, lds, stream, a, err, experts);
}

nh_status launch_mx_tiles(nh_context* ctx, const void* x, nh_dtype dtype, size_t rows, size_t k, uint8_t* out,
                          uint8_t* token_scales, uint64_t* nonfinite, nh_stream stream, nh_error* err) {
    MxQuantizeTilesArgs q{x, out, token_scales, nonfinite, (int64_t)rows, (int32_t)k, (int)mx_k_tiles(k),
                          (int)mx_k_pieces(k), dtype, token_scales ? 1 : 0, rows * k >= (4u << 20) ? 1 : 0};
    return launch(ctx, K_MX_QUANTIZE_TILES, (unsigned)((rows + 15) / 16 * q.kq), 256, 0, stream, q, err);
}

nh_status launch_mx_gemm(nh_context* ctx, const uint8_t* a, const uint8_t* w, const float* bias, size_t m, size_t n,
                         size_t k, void* out, nh_dtype out_dtype, nh_stream stream, nh_error* err) {
    // Tiles by time: a round of workgroups takes so many us per K tile with every
    // CU at its full number of them, or with one per CU at most, and so many for
    // its outputs.  From 72 products of 80..2048 rows, 1024..21504 columns, K
    // 512..8192, each with every tile; the choice is within 8% of the best of
    // them but where few tiles meet a long K (2048 x 8192 -> 4096: 256 / 128 / 64
    // tiles take 68.5 / 57.5 / 72.9 us; 8192 -> 8192 76 / 98 / 127; 300 x 8192 ->
    // 4096 62 / 37 / 21).
    struct Tile {
        KernelId id;
        int b, threads, ks, stages, per_cu;
        double full, one, store;
    };
    static const Tile kTiles[] = {{K_MX_GEMM_256, 256, 512, 1, 4, 1, 0.8, 0.8, 6.0},
                                  {K_MX_GEMM_128, 128, 256, 1, 4, 2, 0.72, 0.42, 3.4},
                                  {K_MX_GEMM_64, 64, 256, 4, 2, 2, 0.31, 0.18, 1.1}};
    const size_t cus = (size_t)ctx->cu_count;
    const double kt = (double)mx_k_tiles(k);
    const Tile* t = nullptr;
    double least = 0.0;
    for (const Tile& c : kTiles) {
        const size_t tiles = ((m + c.b - 1) / c.b) * ((n + c.b - 1) / c.b), round = cus * c.per_cu, rest = tiles % round;
        const double time = (double)(tiles / round) * (kt * c.full + c.store) +
                            (rest == 0 ? 0.0 : kt * (rest <= cus ? c.one : c.full) + c.store);
        if (!t || time < least) {
            t = &c;
            least = time;
        }
    }
    MxGemmArgs g{a, w, bias, out, (int)m, (int)n, (int)mx_k_tiles(k), (int)mx_k_pieces(k), (int)((m + t->b - 1) / t->b),
                 (int)((n + t->b - 1) / t->b), out_dtype, 0};
    // the ring's stages, the pieces of scales that they span (mx_gemm_pieces), a spare KiB
    const size_t tiles = (size_t)g.tiles_m * g.tiles_n, row_tiles = (size_t)2 * t->b / 16;
    const size_t pieces = t->ks == 4 ? t->stages : t->stages / 2 + 1;
    const size_t lds = row_tiles * ((size_t)t->stages * t->ks * 1024 + pieces * 256) + 1024;
    const unsigned grid = (unsigned)std::min(tiles, cus * t->per_cu);
    return launch(ctx, t->id, grid, (unsigned)t->threads, lds, stream, g, err);
}

}  // namespace

extern "C" {

nh_status nh_quantize_rows_mxfp4(nh_context* ctx, const void* x, nh_dtype dtype, size_t rows, size_t cols,
                                 uint8_t* codes, uint8_t* scales, uint64_t* nonfinite, nh_stream stream, nh_error* err) {
    clear_error(err);
    nh_status st;
    if ((st = check_dtype(dtype, err)) || (st = check_mx_rows(rows, cols, err))) return st;
    if (rows != 0 && cols != 0 && (st = check_given({x, codes, scales}, err))) return st;
    if ((st = bind_device(ctx, err))) return st;
    if (rows == 0 || cols == 0) return NH_OK;
    const int64_t row_units = (int64_t)mx_row_blocks(cols) * 4, units = (int64_t)rows * row_units;
    MxQuantizeArgs a{x, codes, scales, nonfinite, units, (int64_t)rows, (uint32_t)cols, (uint32_t)row_units, dtype,
                     cols % kMxBlock == 0 ? 1 : 0};
    return launch(ctx, K_MX_QUANTIZE, mx_unit_grid(units), 256, 0, stream, a, err);
}

nh_status nh_dequantize_mxfp4(nh_context* ctx, const uint8_t* codes, const uint8_t* scales, size_t rows, size_t cols,
                              void* out, nh_dtype out_dtype, nh_stream stream, nh_error* err) {
    clear_error(err);
    nh_status st;
    if ((st = check_dtype(out_dtype, err)) || (st = check_mx_rows(rows, cols, err))) return st;
    if (rows != 0 && cols != 0 && (st = check_given({codes, scales, out}, err))) return st;
    if ((st = bind_device(ctx, err))) return st;
    if (rows == 0 || cols == 0) return NH_OK;
    const int64_t row_units = (int64_t)mx_row_blocks(cols) * 4, units = (int64_t)rows * row_units;
    MxDequantizeArgs a{codes, scales, out, units, (uint32_t)cols, (uint32_t)row_units, out_dtype,
                       cols % kMxBlock == 0 ? 1 : 0};
    return launch(ctx, K_MX_DEQUANTIZE, mx_unit_grid(units), 256, 0, stream, a, err);
}

size_t nh_tiled_mxfp4_weights_bytes(size_t n, size_t k) {
    if (n == 0 || k == 0 || n > (1ull << 40) || k > (1ull << 40) || (n >> 20) * (k >> 20) >= (1ull << 20)) return 0;
    return (size_t)mx_tiled_bytes(n, k);
}

nh_status nh_tile_weights_mxfp4(nh_context* ctx, const uint8_t* codes, const uint8_t* scales, size_t n, size_t k,
                                uint8_t* tiled, size_t tiled_len, nh_stream stream, nh_error* err) {
    clear_error(err);
    const size_t need = nh_tiled_mxfp4_weights_bytes(n, k);
    if (need == 0) return set_error(err, NH_INVALID_SHAPE, "invalid weight shape n=%zu k=%zu", n, k);
    if (n >= (1u << 31) || k > (size_t)kMaxGrid - 128) return set_error(err, NH_UNSUPPORTED, "n and k must be < 2^31");
    if (tiled_len != need) return mismatch(err, "tiled", need, tiled_len);
    if (!aligned16(tiled)) return set_error(err, NH_UNSUPPORTED, "tiled must be 16-byte aligned");
    nh_status st;
    if ((st = check_given({codes, scales, tiled}, err)) || (st = bind_device(ctx, err))) return st;
    const int kq = (int)mx_k_pieces(k);
    MxTileArgs a{codes, scales, tiled, (int64_t)((n + 15) / 16) * kq * 64, (int64_t)n, (int32_t)k, (int)mx_k_tiles(k), kq, 0};
    const int64_t grid = std::min<int64_t>((a.lanes + 255) / 256, 1 << 20);
    return launch(ctx, K_MX_TILE, (unsigned)grid, 256, 0, stream, a, err);
}

int nh_supports_linear_mxfp4(size_t m, size_t n, size_t k) {
    // K up to 2^17 keeps 16 row tiles of codes and scales within a 32-bit
    // buffer offset, m n below 2^40 the output tiles and their stages within 31 bits;
    // the rows' quantization has a workgroup of 256 per 16 rows and 512 columns
    return m > 0 && n > 0 && k > 0 && m < (1u << 24) && n < (1u << 28) && k <= (1u << 17) &&
           (uint64_t)m * n < (1ull << 40) && (uint64_t)m * k < (1ull << 38) &&
           launchable((m + 15) / 16 * mx_k_pieces(k), 256);
}

size_t nh_linear_mxfp4_workspace_size(size_t m, size_t n, size_t k) {
    if (!nh_supports_linear_mxfp4(m, n, k)) return 0;
    if (m <= kMxRowsMax && k <= kMxRowsMaxK) return 0;
    return align256((size_t)mx_tiled_bytes(m, k));  // the token form of the rows is no larger
}

nh_status nh_linear_mxfp4(nh_context* ctx, const void* x, nh_dtype x_dtype, const uint8_t* w, const float* bias,
                          size_t m, size_t n, size_t k, void* out, nh_dtype out_dtype, void* workspace,
                          size_t workspace_bytes, uint64_t* nonfinite, nh_stream stream, nh_error* err) {
    clear_error(err);
    if (n == 0 || k == 0) return set_error(err, NH_INVALID_SHAPE, "invalid linear shape k=%zu n=%zu", k, n);
    if (m == 0) return set_error(err, NH_INVALID_ROW_COUNT, "row_count must be non-zero, got 0");
    nh_status st;
    if ((st = check_dtype(x_dtype, err)) || (st = check_dtype(out_dtype, err))) return st;
    if (!nh_supports_linear_mxfp4(m, n, k))
        return set_error(err, NH_UNSUPPORTED, "shape m=%zu n=%zu k=%zu outside the gfx950 envelope (k <= 131072, "
                         "m < 2^24, n < 2^28, m * n < 2^40, ceil(m / 16) * ceil(k / 512) < 2^24)", m, n, k);
    if ((st = check_given({x, w, out}, err))) return st;
    if (!aligned16(w)) return set_error(err, NH_UNSUPPORTED, "w must be 16-byte aligned");
    const size_t need = nh_linear_mxfp4_workspace_size(m, n, k);
    if (need && (!workspace || workspace_bytes < need)) return mismatch(err, "workspace", need, workspace_bytes);
    if (need && !aligned16(workspace)) return set_error(err, NH_UNSUPPORTED, "workspace must be 16-byte aligned");
    // the one-launch form stores outputs while other workgroups still read x
    if (overlap(out, m * n * (out_dtype == NH_BF16 ? 2 : 4), x, m * k * (x_dtype == NH_BF16 ? 2 : 4)))
        return set_error(err, NH_INVALID_PARAMS, "out must not overlap x");
    if ((st = bind_device(ctx, err))) return st;
    MxStreamArgs a{};
    a.w = w;
    a.bias = bias;
    a.out = out;
    a.M = (int)m;
    a.N = (int)n;
    a.K = (int)k;
    a.kt = (int)mx_k_tiles(k);
    a.kq = (int)mx_k_pieces(k);
    a.x_dtype = x_dtype;
    a.out_dtype = out_dtype;
    a.gather_div = 1;
    a.row_parts = 1;
    const unsigned cus = (unsigned)ctx->cu_count;
    if (need == 0) {
        a.x = x;
        a.nonfinite = nonfinite;
        // rows that start at 16-byte boundaries and hold whole blocks load
        // without a branch, up to what fits the registers
        const bool straight = k % kMxBlock == 0 && aligned16(x) && k <= (x_dtype == NH_BF16 ? 8192 : 4096);
        const KernelId id = !straight ? K_MX_ANY_2 : x_dtype == NH_BF16 ? K_MX_BF16_2 : K_MX_F32_2;
        return launch_mx_stream(ctx, id, a, m, false, cus, 1, stream, err);
    }
    uint8_t* ws = (uint8_t*)workspace;
    if (mx_streams(m, n, k)) {
        uint8_t* scales = ws + m * mx_token_codes(k);
        if ((st = launch_mx_tiles(ctx, x, x_dtype, m, k, ws, scales, nonfinite, stream, err))) return st;
        a.xcodes = ws;
        a.xscales = scales;
        return launch_mx_stream(ctx, K_MX_TOK2, a, m, false, cus, 1, stream, err);
    }
    if ((st = launch_mx_tiles(ctx, x, x_dtype, m, k, ws, nullptr, nonfinite, stream, err))) return st;
    return launch_mx_gemm(ctx, ws, w, bias, m, n, k, out, out_dtype, stream, err);
}

}  // extern "C"

// Workgroups (of 1024) that the MoE layer's prep launch routes and quantizes with.
// One that routes alone, 16 tokens at a time, also sorts the routes, every thread
// against all of them, while that takes less than a launch of its own (layers of
// 128 small experts: 8 tokens with 6 routes each 23.3 us, 24.6 with the launch; 16
// with 4 23.6 and 24.4; 8 with 16 32.9 and 31.4; 32 with 6, in two turns, 35.5 and
// 28.5).
static bool mx_moe_permutes(size_t T, size_t R) { return T <= 16 && R <= 64; }
static size_t mx_moe_route_blocks(size_t T, size_t R) { return mx_moe_permutes(T, R) ? 1 : (T + 15) / 16; }
static size_t mx_moe_quantize_blocks(size_t T, size_t H) { return ((T + 15) / 16 * mx_k_pieces(H) + 3) / 4; }

// Workspace of the MoE layer, 256-byte aligned fields; false: sizes overflow.
static bool mx_moe_layout(size_t T, size_t H, size_t I, size_t E, size_t k, size_t off[11]) {
    size_t R, t;
    if (T == 0 || H == 0 || I == 0 || E == 0 || k == 0 || !mul_ok(T, k, &R) || R >= (1ull << 31) || H > (1u << 24) ||
        I > (1u << 24) || E > (1u << 24) || !mul_ok(R * 4, std::max(H, I), &t) || t >= (1ull << 60))
        return false;
    size_t cur = 0;
    auto take = [&](size_t bytes) {
        const size_t o = cur;
        cur += align256(bytes);
        return o;
    };
    off[0] = take(R * 4);                        // indices
    off[1] = take(R * 4);                        // weights
    off[2] = take((E + 1) * 4);                  // offsets
    off[3] = take(R * 4);                        // perm
    off[4] = take(R * 4);                        // pos
    off[5] = take(T * mx_token_codes(H));        // x in MXFP4, token form
    off[6] = take(T * mx_token_scales(H));
    off[7] = take(R * mx_token_codes(I));        // h in MXFP4, token form by slot
    off[8] = take(R * mx_token_scales(I));
    off[9] = take(R * H * 4);                    // down output per slot (f32)
    off[10] = cur;
    return true;
}

extern "C" {

int nh_supports_moe_forward_mxfp4(size_t tokens, size_t hidden, size_t inter, size_t experts, size_t top_k) {
    size_t off[11];
    if (!mx_moe_layout(tokens, hidden, inter, experts, top_k, off) || top_k > experts) return 0;
    // one launch routes and quantizes; a non-finite word has 38 bits for an index into x or h
    const uint64_t routes = (uint64_t)tokens * top_k;
    return experts <= 1024 && top_k <= 64 && hidden <= 8192 && inter <= 8192 &&
           launchable(mx_moe_route_blocks(tokens, routes) + mx_moe_quantize_blocks(tokens, hidden), 1024) &&
           routes * inter < (1ull << 38);
}

size_t nh_moe_forward_mxfp4_workspace_size(size_t tokens, size_t hidden, size_t inter, size_t experts, size_t top_k) {
    size_t off[11];
    return mx_moe_layout(tokens, hidden, inter, experts, top_k, off) ? off[10] : 0;
}

void nh_moe_mxfp4_workspace_layout(size_t tokens, size_t hidden, size_t inter, size_t experts, size_t top_k,
                                   size_t offsets_out[5]) {
    size_t off[11] = {};
    mx_moe_layout(tokens, hidden, inter, experts, top_k, off);
    for (int i = 0; i < 5; ++i) offsets_out[i] = off[i];
}

nh_status nh_moe_forward_mxfp4(nh_context* ctx, const void* x, nh_dtype x_dtype, const float* logits, size_t tokens,
                               size_t hidden, size_t inter, size_t experts, size_t top_k, int renormalize,
                               float scaling, const uint8_t* w_up, const uint8_t* w_down, const nh_moe_biases* biases,
                               const float* shared, void* out, nh_dtype out_dtype, void* workspace,
                               size_t workspace_bytes, uint64_t* nonfinite, nh_stream stream, nh_error* err) {
    clear_error(err);
    if (tokens == 0) return set_error(err, NH_INVALID_ROW_COUNT, "row_count must be non-zero, got 0");
    size_t off[11];
    if (top_k > experts || !mx_moe_layout(tokens, hidden, inter, experts, top_k, off))
        return set_error(err, NH_INVALID_SHAPE, "invalid MoE shape");
    if (biases && (biases->shared_up || biases->shared_down))
        return set_error(err, NH_INVALID_PARAMS, "shared expert biases given without a shared expert");
    nh_status st;
    if ((st = check_dtype(x_dtype, err)) || (st = check_dtype(out_dtype, err))) return st;
    if (!nh_supports_moe_forward_mxfp4(tokens, hidden, inter, experts, top_k))
        return set_error(err, NH_UNSUPPORTED, "MoE shape outside the gfx950 envelope (experts <= 1024, top_k <= 64, "
                         "hidden and inter <= 8192, ceil(tokens / 16) * (1 + ceil(hidden / 512) / 4) < 2^22, "
                         "tokens * top_k * inter < 2^38)");
    if ((st = check_given({x, logits, w_up, w_down, out}, err))) return st;
    if (!workspace || workspace_bytes < off[10]) return mismatch(err, "workspace", off[10], workspace_bytes);
    if (!aligned16(workspace) || !aligned16(w_up) || !aligned16(w_down))
        return set_error(err, NH_UNSUPPORTED, "weights and workspace must be 16-byte aligned");
    if ((st = bind_device(ctx, err))) return st;
    uint8_t* ws = (uint8_t*)workspace;
    int32_t *idx = (int32_t*)(ws + off[0]), *offsets = (int32_t*)(ws + off[2]), *perm = (int32_t*)(ws + off[3]),
            *pos = (int32_t*)(ws + off[4]);
    float *wts = (float*)(ws + off[1]), *d = (float*)(ws + off[9]);
    const size_t R = tokens * top_k;
    // routing beside the tokens' quantization; the routes of a few tokens are
    // sorted in the same launch (one workgroup routes 16 tokens at a time)
    MxMoePrepArgs prep{};
    prep.q = MxQuantizeTilesArgs{x, ws + off[5], ws + off[6], nonfinite, (int64_t)tokens, (int32_t)hidden,
                                 (int)mx_k_tiles(hidden), (int)mx_k_pieces(hidden), x_dtype, 1, 0};
    prep.r.scores = logits;
    prep.r.indices = idx;
    prep.r.weights = wts;
    prep.r.tokens = (int)tokens;
    prep.r.experts = (int)experts;
    prep.r.top_k = (int)top_k;
    prep.r.renormalize = renormalize ? 1 : 0;
    prep.r.scaling = scaling;
    prep.p = PermuteArgs{idx, offsets, perm, pos, (int)R, (int)experts};
    prep.permute = mx_moe_permutes(tokens, R) ? 1 : 0;
    prep.route_blocks = (int)mx_moe_route_blocks(tokens, R);
    if ((st = launch(ctx, K_MX_MOE_PREP, (unsigned)(prep.route_blocks + mx_moe_quantize_blocks(tokens, hidden)), 1024, 0,
                     stream, prep, err)))
        return st;
    if (!prep.permute && (st = nh_moe_permute(ctx, idx, tokens, top_k, experts, offsets, perm, pos, stream, err))) return st;
    // As many workgroups per expert as give every CU one when the routes reach
    // as many experts as evenly spread ones do and three standard deviations
    // more (a few past the CUs cost a second round: 8 tokens over 128 experts in
    // 6 parts each took 67 or 82 us by the input); slots packed onto the
    // experts with routes where a tenth has none.
    const double live = expected_experts(experts, R), load = (double)R / (double)experts, q = std::exp(-load);
    const double var = (double)experts * (q - (1.0 + load) * q * q);
    const double most = std::min({(double)experts, (double)R, live + 3.0 * std::sqrt(std::max(0.0, var))});
    // An expert's passes go to workgroups of their own where the mean expert has
    // several (700 tokens, 2 of 8 experts, 4096 x 1792: 97 us one after another, 85).
    auto plan = [&](MxStreamArgs& a, size_t n, size_t k, unsigned* parts, unsigned* slots) {
        a.N = (int)n;
        a.K = (int)k;
        a.kt = (int)mx_k_tiles(k);
        a.kq = (int)mx_k_pieces(k);
        const double pass = mx_pass_rows(tokens, a.kt);
        a.row_parts = load <= pass ? 1 : (int)std::min(std::ceil((load + 2.0 * std::sqrt(load)) / pass), 32.0);
        *parts = (unsigned)std::max(1.0, (double)ctx->cu_count / (most * a.row_parts));
        *slots = (unsigned)(a.compact ? std::min(experts, R) : experts) * (unsigned)a.row_parts;
    };
    unsigned parts, slots;
    MxStreamArgs a{};
    a.offsets = offsets;
    a.experts = (int)experts;
    a.compact = live < 0.9 * (double)experts ? 1 : 0;
    a.xcodes = ws + off[5];
    a.xscales = ws + off[6];
    a.w = w_up;
    a.bias = biases ? biases->up : nullptr;
    a.hcodes = ws + off[7];
    a.hscales = ws + off[8];
    a.nonfinite = nonfinite;
    a.nonfinite_stage = kStageIntermediate;
    a.perm = perm;
    a.gather_div = (int)top_k;
    a.M = (int)R;
    plan(a, inter, hidden, &parts, &slots);
    if ((st = launch_mx_stream(ctx, K_MX_REQUANT2, a, tokens, true, parts, slots, stream, err)))
        return st;
    a.xcodes = ws + off[7];
    a.xscales = ws + off[8];
    a.w = w_down;
    a.bias = biases ? biases->down : nullptr;
    a.hcodes = a.hscales = nullptr;
    a.perm = nullptr;
    a.out = d;
    a.out_dtype = DT_F32;
    plan(a, hidden, inter, &parts, &slots);
    if ((st = launch_mx_stream(ctx, K_MX_TOK2, a, tokens, false, parts, slots, stream, err))) return st;
    return nh_moe_combine_shared(ctx, d, pos, wts, shared, tokens, top_k, hidden, out, out_dtype, stream, err);
}

// ---- load balance of the router ---------------------------------------------
}  // extern "C"

namespace {

struct BalancePlan {
    int chunk, chunks, group;
    size_t part_n, seq_loss, arrived, bytes;  // workspace offsets and size
};

bool plan_balance(size_t sequences, size_t tokens, size_t experts, BalancePlan* p) {
    // every workgroup walks the offsets, 64 at a time
    if (sequences == 0 || experts == 0 || sequences > 16384 || tokens >= (1u << 30) || experts > 1024 ||
        tokens * experts >= (1ull << 40))
        return false;
    // a chunk per CU of 256, of 64 tokens at least
    p->chunk = (int)std::max<size_t>(64, (tokens + 255) / 256);
    p->chunks = (int)(tokens / (size_t)p->chunk + sequences);  // each sequence's last one may be short
    p->group = 1;
    while (4 * p->group < (int)experts && p->group < 64) p->group *= 2;
    const size_t part = align256((size_t)p->chunks * experts * 4);
    p->part_n = part;
    p->seq_loss = 2 * part;
    p->arrived = p->seq_loss + align256(sequences * sizeof(double));
    p->bytes = p->arrived + 256;
    return true;
}

nh_status check_balance(size_t sequences, const int32_t* seq_offsets, size_t tokens, size_t experts, size_t top_k,
                        float coefficient, BalancePlan* p, nh_error* err) {
    if (experts == 0 || top_k == 0 || sequences == 0 || (!seq_offsets && sequences != 1))
        return set_error(err, NH_INVALID_SHAPE, "invalid balance shape sequences=%zu experts=%zu top_k=%zu", sequences,
                         experts, top_k);
    if (!std::isfinite(coefficient)) return set_error(err, NH_INVALID_PARAMS, "coefficient must be finite");
    if (!nh_supports_moe_balance_loss(sequences, tokens, experts, top_k))
        return set_error(err, NH_UNSUPPORTED, "device balance needs experts <= 1024, sequences <= 16384, "
                         "tokens < 2^30 and tokens * top_k < 2^31");
    plan_balance(sequences, tokens, experts, p);
    return NH_OK;
}

}  // namespace

extern "C" {

int nh_supports_moe_balance_loss(size_t sequences, size_t tokens, size_t experts, size_t top_k) {
    BalancePlan p;
    return plan_balance(sequences, tokens, experts, &p) && top_k > 0 && top_k <= 1024 && tokens * top_k < (1ull << 31);
}

size_t nh_moe_balance_loss_workspace_size(size_t sequences, size_t tokens, size_t experts) {
    BalancePlan p;
    return plan_balance(sequences, tokens, experts, &p) ? p.bytes : 0;
}

nh_status nh_moe_balance_loss(nh_context* ctx, const float* logits, const int32_t* indices, const int32_t* seq_offsets,
                              size_t sequences, size_t tokens, size_t experts, size_t top_k, int softmax,
                              float coefficient, int32_t* counts, float* loss, void* workspace, size_t workspace_bytes,
                              nh_stream stream, nh_error* err) {
    clear_error(err);
    BalancePlan p;
    nh_status st = check_balance(sequences, seq_offsets, tokens, experts, top_k, coefficient, &p, err);
    if (st) return st;
    if ((st = check_given({counts, loss}, err))) return st;
    if (tokens != 0 && (st = check_given({logits, indices}, err))) return st;
    if (!workspace || workspace_bytes < p.bytes) return mismatch(err, "workspace", p.bytes, workspace_bytes);
    if (!aligned16(workspace)) return set_error(err, NH_UNSUPPORTED, "workspace must be 16-byte aligned");
    if ((st = bind_device(ctx, err))) return st;
    uint8_t* ws = (uint8_t*)workspace;
    BalanceArgs a{};
    a.logits = logits;
    a.indices = indices;
    a.seq = seq_offsets;
    a.counts = counts;
    a.loss = loss;
    a.part_p = (float*)ws;
    a.part_n = (int32_t*)(ws + p.part_n);
    a.seq_loss = (double*)(ws + p.seq_loss);
    a.arrived = (uint32_t*)(ws + p.arrived);
    a.tokens = (int)tokens;
    a.experts = (int)experts;
    a.top_k = (int)top_k;
    a.sequences = (int)sequences;
    a.chunk = p.chunk;
    a.chunks = p.chunks;
    a.softmax = softmax ? 1 : 0;
    a.coefficient = coefficient;
    a.group = p.group;
    // a few rows and routes, one sequence: one workgroup and launch (64 x 128 5.8 us,
    // 8.3 in two; 192 x 128 8.4 and 9.1, 256 x 128 10.3 and 9.1; 4096 x 8 10.1 and 10.7
    // with 2 routes each, 13.6 and 10.5 with 8; 16384 x 1 24 and 27, 32768 x 1 44 and 27)
    a.single = sequences == 1 && tokens * experts <= 256 * 128 && tokens * top_k <= 16384 ? 1 : 0;
    const size_t lds = 17 * experts * 4 + 256;
    if (a.single) return launch(ctx, K_BALANCE_PARTIAL, 1, 1024, lds, stream, a, err);
    if ((st = launch(ctx, K_BALANCE_PARTIAL, (unsigned)p.chunks, 1024, lds, stream, a, err))) return st;
    return launch(ctx, K_BALANCE_REDUCE, (unsigned)sequences, 1024, 128 + 1024 * 12, stream, a, err);
}

nh_status nh_moe_balance_loss_backward(nh_context* ctx, const float* logits, const int32_t* counts,
                                       const int32_t* seq_offsets, size_t sequences, size_t tokens, size_t experts,
                                       size_t top_k, int softmax, float coefficient, const float* dloss, float* dlogits,
                                       nh_stream stream, nh_error* err) {
    clear_error(err);
    BalancePlan p;
    nh_status st = check_balance(sequences, seq_offsets, tokens, experts, top_k, coefficient, &p, err);
    if (st) return st;
    if (tokens != 0 && (st = check_given({logits, counts, dloss, dlogits}, err))) return st;
    if ((st = bind_device(ctx, err))) return st;
    if (tokens == 0) return NH_OK;
    BalanceArgs a{};
    a.logits = logits;
    a.seq = seq_offsets;
    a.counts = const_cast<int32_t*>(counts);
    a.dloss = dloss;
    a.dlogits = dlogits;
    a.tokens = (int)tokens;
    a.experts = (int)experts;
    a.top_k = (int)top_k;
    a.sequences = (int)sequences;
    a.softmax = softmax ? 1 : 0;
    a.coefficient = coefficient;
    a.group = p.group;
    // chunks for four workgroups of four waves per CU, of 32 tokens at least
    a.chunk = (int)std::max<size_t>(32, (tokens + 4 * (size_t)ctx->cu_count - 1) / (4 * (size_t)ctx->cu_count));
    a.chunks = (int)(tokens / (size_t)a.chunk + sequences);
    a.padding = seq_offsets ? 64 : 0;
    return launch(ctx, K_BALANCE_BACKWARD, (unsigned)(a.chunks + a.padding), 256, 0, stream, a, err);
}

}  // extern "C"
