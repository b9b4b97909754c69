// Which operands of the rows by expert and of the adapters must not share bytes: the
// device entry points and their host twins refuse the same calls.
#pragma once
#include "../runtime/nh_runtime.h"

namespace nh {

inline size_t bytes_of(nh_dtype d) { return d == NH_BF16 ? 2 : 4; }

inline nh_status dispatch_apart(const void* x, nh_dtype x_dtype, const int32_t* pos, const float* weights, size_t tokens,
                                size_t top_k, size_t hidden, size_t slots, void* rows, nh_dtype rows_dtype, nh_error* err) {
    const size_t routes = tokens * top_k * 4;
    if (apart({{rows, slots * hidden * bytes_of(rows_dtype)}},
              {{x, tokens * hidden * bytes_of(x_dtype)}, {pos, routes}, {weights, routes}}))
        return NH_OK;
    return set_error(err, NH_INVALID_PARAMS, "rows must not overlap another operand");
}

inline nh_status dispatch_backward_apart(const void* drows, nh_dtype rows_dtype, const void* x, nh_dtype x_dtype,
                                         const int32_t* pos, const float* weights, size_t tokens, size_t top_k,
                                         size_t hidden, size_t slots, void* dx, float* dweights, nh_error* err) {
    const size_t token_bytes = tokens * hidden * bytes_of(x_dtype), routes = tokens * top_k * 4;
    if (apart({{dx, token_bytes}, {dweights, routes}},
              {{drows, slots * hidden * bytes_of(rows_dtype)}, {dweights ? x : nullptr, token_bytes}, {pos, routes}, {weights, routes}}))
        return NH_OK;
    return set_error(err, NH_INVALID_PARAMS, "dx and dweights must not overlap another operand");
}

inline nh_status combine_rows_apart(const void* rows, nh_dtype rows_dtype, const int32_t* pos, const float* weights,
                                    const void* shared, size_t tokens, size_t top_k, size_t hidden, size_t slots, void* out,
                                    nh_dtype out_dtype, nh_error* err) {
    const size_t token_bytes = tokens * hidden * bytes_of(out_dtype), routes = tokens * top_k * 4;
    if (apart({{out, token_bytes}}, {{rows, slots * hidden * bytes_of(rows_dtype)}, {shared != out ? shared : nullptr, token_bytes},
                                     {pos, routes}, {weights, routes}}))
        return NH_OK;
    return set_error(err, NH_INVALID_PARAMS, "out must not overlap another operand, but for shared as a whole");
}

inline nh_status combine_rows_backward_apart(const void* dout, nh_dtype out_dtype, const void* rows, nh_dtype rows_dtype,
                                             const int32_t* pos, const float* weights, size_t tokens, size_t top_k,
                                             size_t hidden, size_t slots, void* drows, float* dweights, nh_error* err) {
    const size_t row_bytes = slots * hidden * bytes_of(rows_dtype), routes = tokens * top_k * 4;
    if (apart({{drows, row_bytes}, {dweights, routes}},
              {{dout, tokens * hidden * bytes_of(out_dtype)}, {dweights && rows != drows ? rows : nullptr, row_bytes},
               {pos, routes}, {weights, routes}}))
        return NH_OK;
    return set_error(err, NH_INVALID_PARAMS, "drows and dweights must not overlap another operand, but for rows as a whole");
}

inline nh_status lora_apart(const void* x, nh_dtype x_dtype, const int32_t* adapter_ids, const void* a, const void* b,
                            nh_dtype w_dtype, const float* scales, size_t m, size_t n, size_t k, size_t rank,
                            size_t adapters, const void* base, void* out, nh_dtype out_dtype, float* h_out, nh_error* err) {
    const size_t out_bytes = m * n * bytes_of(out_dtype), matrix = adapters * rank * bytes_of(w_dtype);
    if (apart({{out, out_bytes}, {h_out, m * rank * 4}},
              {{x, m * k * bytes_of(x_dtype)}, {base != out ? base : nullptr, out_bytes}, {adapter_ids, m * 4}, {a, matrix * k},
               {b, matrix * n}, {scales, adapters * 4}}))
        return NH_OK;
    return set_error(err, NH_INVALID_PARAMS, "out and h_out must not overlap another operand, but for base as a whole");
}

inline nh_status lora_backward_apart(const void* x, nh_dtype x_dtype, const int32_t* adapter_ids, const void* a,
                                     const void* b, nh_dtype w_dtype, const float* scales, const float* h, const void* dout,
                                     nh_dtype dout_dtype, size_t m, size_t n, size_t k, size_t rank, size_t adapters,
                                     const void* dx_base, void* dx, float* da, float* db, nh_error* err) {
    const size_t x_bytes = m * k * bytes_of(x_dtype), matrix = adapters * rank;
    if (apart({{dx, x_bytes}, {da, matrix * k * 4}, {db, matrix * n * 4}},
              {{x, x_bytes}, {dx_base != dx ? dx_base : nullptr, x_bytes}, {dout, m * n * bytes_of(dout_dtype)}, {adapter_ids, m * 4},
               {a, matrix * k * bytes_of(w_dtype)}, {b, matrix * n * bytes_of(w_dtype)}, {scales, adapters * 4}, {h, m * rank * 4}}))
        return NH_OK;
    return set_error(err, NH_INVALID_PARAMS, "dx, da and db must not overlap another operand, but for dx_base as a whole");
}

}  // namespace nh
