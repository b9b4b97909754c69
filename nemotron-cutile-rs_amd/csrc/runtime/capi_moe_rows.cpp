// Device entry points of the rows by expert: validate on the host, then enqueue.
#include <algorithm>
#include <cstdint>

#include "../host/adapters_operands.h"

using namespace nh;

namespace {

nh_status check_rows(nh_dtype token, nh_dtype row, size_t tokens, size_t top_k, size_t hidden, size_t slots,
                     nh_error* err) {
    nh_status st;
    if (top_k == 0 || hidden == 0)
        return set_error(err, NH_INVALID_SHAPE, "invalid rows shape top_k=%zu hidden=%zu", top_k, hidden);
    if ((st = check_dtype(token, err)) || (st = check_dtype(row, err))) return st;
    if (!nh_supports_moe_rows(tokens, top_k, hidden, slots))
        return set_error(err, NH_UNSUPPORTED, "device rows need tokens * top_k, slots and hidden < 2^31, "
                         "tokens * hidden and slots * hidden < 2^40");
    return NH_OK;
}

// One workgroup per token; 16 bytes of a row per thread and turn, as many threads
// as take it in the fewest turns of at most 512.
// Rows go past the caches from 64 MiB on, but for a gather with the weights' gradients,
// which reads them twice.  Through them and past them, us, 2688 wide, 6 routes, bf16,
// rows of 32, 64 and 264 MiB: dispatch 9.5, 8.6; 21, 15; 74, 56.  Combine 9.1, 9.8; 18.0,
// 17.6; 63, 62, with the dispatch of the same rows 19, 18; 36, 33; 158, 118.  Combine
// backward 21, 18; 35, 30; 124, 113.  Dispatch backward with the weights' gradients 15, 18;
// 28, 31; 92, 111.
nh_status launch_rows(nh_context* ctx, KernelId first, MoeRowsArgs a, nh_dtype token, nh_dtype row, size_t tokens,
                      nh_stream stream, nh_error* err) {
    const KernelId id = (KernelId)(first + (token == NH_BF16 ? 2 : 0) + (row == NH_BF16 ? 1 : 0));
    const size_t v = row == NH_BF16 ? 8 : 4, vectors = ((size_t)a.hidden + v - 1) / v, turns = (vectors + 511) / 512;
    const size_t threads = ((vectors + turns - 1) / turns + 63) / 64 * 64;
    const bool twice = first == K_MOE_GATHER && a.dweights;
    a.far = !twice && tokens * (size_t)a.top_k * (size_t)a.hidden * bytes_of(row) >= ((size_t)64 << 20) ? 1 : 0;
    const size_t most = ((1ull << 32) - 1) / threads;  // workgroups of a launch: fewer than 2^32 threads
    for (size_t t0 = 0; t0 < tokens; t0 += most) {
        a.token0 = (int64_t)t0;
        const nh_status st = launch(ctx, id, (unsigned)std::min(most, tokens - t0), (unsigned)threads, 0, stream, a, err);
        if (st) return st;
    }
    return NH_OK;
}

}  // namespace

extern "C" {

int nh_supports_moe_rows(size_t tokens, size_t top_k, size_t hidden, size_t slots) {
    size_t routes;
    return top_k > 0 && hidden > 0 && hidden <= (size_t)kMaxGrid && slots <= (size_t)kMaxGrid && tokens <= (size_t)kMaxGrid &&
           mul_ok(tokens, top_k, &routes) && routes <= (size_t)kMaxGrid && tokens * hidden < (1ull << 40) &&
           slots * hidden < (1ull << 40);
}

nh_status nh_moe_dispatch(nh_context* ctx, const void* x, nh_dtype x_dtype, const int32_t* pos, const float* weights,
                          size_t tokens, size_t top_k, size_t hidden, size_t slots, void* rows, nh_dtype rows_dtype,
                          nh_stream stream, nh_error* err) {
    clear_error(err);
    nh_status st = check_rows(x_dtype, rows_dtype, tokens, top_k, hidden, slots, err);
    if (st) return st;
    if (tokens != 0 && slots != 0 && (st = check_given({x, pos, rows}, err))) return st;
    if ((st = dispatch_apart(x, x_dtype, pos, weights, tokens, top_k, hidden, slots, rows, rows_dtype, err)) ||
        (st = bind_device(ctx, err)))
        return st;
    if (tokens == 0 || slots == 0) return NH_OK;
    MoeRowsArgs a{};
    a.tokens = x;
    a.pos = pos;
    a.weights = weights;
    a.rows_out = rows;
    a.slots = (int64_t)slots;
    a.top_k = (int)top_k;
    a.hidden = (int)hidden;
    return launch_rows(ctx, K_MOE_SCATTER, a, x_dtype, rows_dtype, tokens, stream, err);
}

nh_status nh_moe_dispatch_backward(nh_context* ctx, const void* drows, nh_dtype rows_dtype, const void* x,
                                   nh_dtype x_dtype, const int32_t* pos, const float* weights, size_t tokens,
                                   size_t top_k, size_t hidden, size_t slots, void* dx, float* dweights,
                                   nh_stream stream, nh_error* err) {
    clear_error(err);
    nh_status st = check_rows(x_dtype, rows_dtype, tokens, top_k, hidden, slots, err);
    if (st) return st;
    if (tokens != 0 && ((st = check_given({pos, dx}, err)) || (slots != 0 && (st = check_given({drows}, err))) ||
                        (dweights && (st = check_given({x}, err)))))
        return st;
    if ((st = dispatch_backward_apart(drows, rows_dtype, x, x_dtype, pos, weights, tokens, top_k, hidden, slots, dx, dweights,
                                      err)) ||
        (st = bind_device(ctx, err)))
        return st;
    if (tokens == 0) return NH_OK;
    MoeRowsArgs a{};
    a.rows_in = drows;
    a.dot = x;
    a.pos = pos;
    a.weights = weights;
    a.out = dx;
    a.dweights = dweights;
    a.slots = (int64_t)slots;
    a.top_k = (int)top_k;
    a.hidden = (int)hidden;
    return launch_rows(ctx, K_MOE_GATHER, a, x_dtype, rows_dtype, tokens, stream, err);
}

nh_status nh_moe_combine_rows(nh_context* ctx, const void* rows, nh_dtype rows_dtype, const int32_t* pos,
                              const float* weights, const void* shared, size_t tokens, size_t top_k, size_t hidden,
                              size_t slots, void* out, nh_dtype out_dtype, nh_stream stream, nh_error* err) {
    clear_error(err);
    nh_status st = check_rows(out_dtype, rows_dtype, tokens, top_k, hidden, slots, err);
    if (st) return st;
    if (tokens != 0 && ((st = check_given({pos, out}, err)) || (slots != 0 && (st = check_given({rows}, err))))) return st;
    if ((st = combine_rows_apart(rows, rows_dtype, pos, weights, shared, tokens, top_k, hidden, slots, out, out_dtype, err)) ||
        (st = bind_device(ctx, err)))
        return st;
    if (tokens == 0) return NH_OK;
    MoeRowsArgs a{};
    a.rows_in = rows;
    a.shared = shared;
    a.pos = pos;
    a.weights = weights;
    a.out = out;
    a.slots = (int64_t)slots;
    a.top_k = (int)top_k;
    a.hidden = (int)hidden;
    return launch_rows(ctx, K_MOE_GATHER, a, out_dtype, rows_dtype, tokens, stream, err);
}

nh_status nh_moe_combine_rows_backward(nh_context* ctx, const void* dout, nh_dtype out_dtype, const void* rows,
                                       nh_dtype rows_dtype, const int32_t* pos, const float* weights, size_t tokens,
                                       size_t top_k, size_t hidden, size_t slots, void* drows, float* dweights,
                                       nh_stream stream, nh_error* err) {
    clear_error(err);
    nh_status st = check_rows(out_dtype, rows_dtype, tokens, top_k, hidden, slots, err);
    if (st) return st;
    if (tokens != 0 && ((st = check_given({dout, pos}, err)) || (slots != 0 && (st = check_given({drows}, err))) ||
                        (dweights && slots != 0 && (st = check_given({rows}, err)))))
        return st;
    if ((st = combine_rows_backward_apart(dout, out_dtype, rows, rows_dtype, pos, weights, tokens, top_k, hidden, slots, drows,
                                          dweights, err)) ||
        (st = bind_device(ctx, err)))
        return st;
    if (tokens == 0) return NH_OK;
    MoeRowsArgs a{};
    a.tokens = dout;
    a.rows_in = rows;
    a.pos = pos;
    a.weights = weights;
    a.rows_out = drows;
    a.dweights = dweights;
    a.slots = (int64_t)slots;
    a.top_k = (int)top_k;
    a.hidden = (int)hidden;
    return launch_rows(ctx, K_MOE_SCATTER, a, out_dtype, rows_dtype, tokens, stream, err);
}

}  // extern "C"
