// Host twins of the rows by expert and of the low-rank adapters (sums in 64 bits).
#include <algorithm>
#include <exception>
#include <vector>

#include "adapters_operands.h"

using namespace nh;

namespace {

float load_f32(const void* x, size_t i, nh_dtype d) {
    return d == NH_BF16 ? bf16_to_f32(((const uint16_t*)x)[i]) : ((const float*)x)[i];
}

void store_f32(void* out, size_t i, float v, nh_dtype d) {
    if (d == NH_BF16)
        ((uint16_t*)out)[i] = f32_to_bf16(v);
    else
        ((float*)out)[i] = v;
}

// Runs the body of a twin; memory that is not there is an error, no exception.
template <class Body>
nh_status guarded(nh_error* err, Body body) {
    try {
        return body();
    } catch (const std::exception&) {  // std::bad_alloc, std::length_error
        return set_error(err, NH_DEVICE_ERROR, "out of host memory");
    }
}

nh_status check_rows(nh_dtype token, nh_dtype row, size_t tokens, size_t top_k, size_t hidden, size_t slots,
                     nh_error* err) {
    size_t t;
    if (top_k == 0 || hidden == 0 || !mul_ok(tokens, top_k, &t) || !mul_ok(tokens, hidden, &t) || !mul_ok(slots, hidden, &t))
        return set_error(err, NH_INVALID_SHAPE, "invalid rows shape top_k=%zu hidden=%zu", top_k, hidden);
    nh_status st;
    if ((st = check_dtype(token, err))) return st;
    return check_dtype(row, err);
}

// rows_out[s] = w v[t], and dw = <rows_in[s], v[t]>.
void scatter(const void* v, nh_dtype vd, const void* rows_in, void* rows_out, nh_dtype rd, const int32_t* pos,
             const float* weights, size_t tokens, size_t top_k, size_t hidden, size_t slots, float* dweights) {
    for (size_t r = 0; r < tokens * top_k; ++r) {
        const bool placed = pos[r] >= 0 && (size_t)pos[r] < slots;
        const size_t t = r / top_k, s = placed ? (size_t)pos[r] : 0;
        double d = 0.0;
        if (placed)
            for (size_t c = 0; c < hidden; ++c) {
                const float x = load_f32(v, t * hidden + c, vd);
                if (dweights) d += (double)load_f32(rows_in, s * hidden + c, rd) * (double)x;
                store_f32(rows_out, s * hidden + c, weights ? weights[r] * x : x, rd);
            }
        if (dweights) dweights[r] = (float)d;
    }
}

// out[t] = shared[t] + sum of w rows[s], and dw = <rows[s], dot[t]>.
void gather(const void* rows, nh_dtype rd, const void* shared, const void* dot, void* out, nh_dtype od,
            const int32_t* pos, const float* weights, size_t tokens, size_t top_k, size_t hidden, size_t slots,
            float* dweights) {
    for (size_t t = 0; t < tokens; ++t) {
        const int32_t* p = pos + t * top_k;
        auto placed = [&](size_t j) { return p[j] >= 0 && (size_t)p[j] < slots; };
        for (size_t j = 0; dweights && j < top_k; ++j) {
            double d = 0.0;
            for (size_t c = 0; placed(j) && c < hidden; ++c)
                d += (double)load_f32(rows, (size_t)p[j] * hidden + c, rd) * (double)load_f32(dot, t * hidden + c, od);
            dweights[t * top_k + j] = (float)d;
        }
        for (size_t c = 0; c < hidden; ++c) {
            double v = shared ? (double)load_f32(shared, t * hidden + c, od) : 0.0;
            for (size_t j = 0; j < top_k; ++j)
                if (placed(j))
                    v += (weights ? (double)weights[t * top_k + j] : 1.0) * (double)load_f32(rows, (size_t)p[j] * hidden + c, rd);
            store_f32(out, t * hidden + c, (float)v, od);
        }
    }
}

nh_status check_lora(size_t m, size_t n, size_t k, size_t rank, size_t adapters, std::initializer_list<nh_dtype> dtypes,
                     nh_error* err) {
    size_t t;
    if (n == 0 || k == 0 || rank == 0 || adapters == 0 || !mul_ok(m, n, &t) || !mul_ok(m, k, &t) || !mul_ok(m, rank, &t) ||
        !mul_ok(rank, n, &t) || !mul_ok(t, adapters, &t) || !mul_ok(rank, k, &t) || !mul_ok(t, adapters, &t))
        return set_error(err, NH_INVALID_SHAPE, "invalid adapter shape k=%zu n=%zu rank=%zu adapters=%zu", k, n, rank, adapters);
    if (m == 0) return set_error(err, NH_INVALID_ROW_COUNT, "row_count must be non-zero, got 0");
    for (nh_dtype d : dtypes)
        if (nh_status st = check_dtype(d, err)) return st;
    return NH_OK;
}

}  // namespace

extern "C" {

nh_status nh_moe_dispatch_host(const void* x, nh_dtype x_dtype, const int32_t* pos, const float* weights, size_t tokens,
                               size_t top_k, size_t hidden, size_t slots, void* rows, nh_dtype rows_dtype,
                               nh_error* err) {
    clear_error(err);
    nh_status st = check_rows(x_dtype, rows_dtype, tokens, top_k, hidden, slots, err);
    if (st) return st;
    if ((tokens != 0 && slots != 0 && (st = check_given({x, pos, rows}, err))) ||
        (st = dispatch_apart(x, x_dtype, pos, weights, tokens, top_k, hidden, slots, rows, rows_dtype, err)))
        return st;
    if (slots != 0) scatter(x, x_dtype, nullptr, rows, rows_dtype, pos, weights, tokens, top_k, hidden, slots, nullptr);
    return NH_OK;
}

nh_status nh_moe_dispatch_backward_host(const void* drows, nh_dtype rows_dtype, const void* x, nh_dtype x_dtype,
                                        const int32_t* pos, const float* weights, size_t tokens, size_t top_k,
                                        size_t hidden, size_t slots, void* dx, float* dweights, nh_error* err) {
    clear_error(err);
    nh_status st = check_rows(x_dtype, rows_dtype, tokens, top_k, hidden, slots, err);
    if (st) return st;
    if (tokens != 0 && ((st = check_given({pos, dx}, err)) || (slots != 0 && (st = check_given({drows}, err))) ||
                        (dweights && (st = check_given({x}, err)))))
        return st;
    if ((st = dispatch_backward_apart(drows, rows_dtype, x, x_dtype, pos, weights, tokens, top_k, hidden, slots, dx, dweights, err)))
        return st;
    gather(drows, rows_dtype, nullptr, x, dx, x_dtype, pos, weights, tokens, top_k, hidden, slots, dweights);
    return NH_OK;
}

nh_status nh_moe_combine_rows_host(const void* rows, nh_dtype rows_dtype, const int32_t* pos, const float* weights,
                                   const void* shared, size_t tokens, size_t top_k, size_t hidden, size_t slots,
                                   void* out, nh_dtype out_dtype, nh_error* err) {
    clear_error(err);
    nh_status st = check_rows(out_dtype, rows_dtype, tokens, top_k, hidden, slots, err);
    if (st) return st;
    if (tokens != 0 && ((st = check_given({pos, out}, err)) || (slots != 0 && (st = check_given({rows}, err))))) return st;
    if ((st = combine_rows_apart(rows, rows_dtype, pos, weights, shared, tokens, top_k, hidden, slots, out, out_dtype, err)))
        return st;
    gather(rows, rows_dtype, shared, nullptr, out, out_dtype, pos, weights, tokens, top_k, hidden, slots, nullptr);
    return NH_OK;
}

nh_status nh_moe_combine_rows_backward_host(const void* dout, nh_dtype out_dtype, const void* rows, nh_dtype rows_dtype,
                                            const int32_t* pos, const float* weights, size_t tokens, size_t top_k,
                                            size_t hidden, size_t slots, void* drows, float* dweights, nh_error* err) {
    clear_error(err);
    nh_status st = check_rows(out_dtype, rows_dtype, tokens, top_k, hidden, slots, err);
    if (st) return st;
    if (tokens != 0 && ((st = check_given({dout, pos}, err)) || (slots != 0 && (st = check_given({drows}, err))) ||
                        (dweights && slots != 0 && (st = check_given({rows}, err)))))
        return st;
    if ((st = combine_rows_backward_apart(dout, out_dtype, rows, rows_dtype, pos, weights, tokens, top_k, hidden, slots, drows,
                                          dweights, err)))
        return st;
    scatter(dout, out_dtype, rows, drows, rows_dtype, pos, weights, tokens, top_k, hidden, slots, dweights);
    return NH_OK;
}

nh_status nh_linear_lora_host(const void* x, nh_dtype x_dtype, const int32_t* adapter_ids, const void* a, const void* b,
                              nh_dtype w_dtype, const float* scales, size_t m, size_t n, size_t k, size_t rank,
                              size_t adapters, const void* base, void* out, nh_dtype out_dtype, float* h_out,
                              nh_error* err) {
    clear_error(err);
    nh_status st;
    if ((st = check_lora(m, n, k, rank, adapters, {x_dtype, w_dtype, out_dtype}, err)) ||
        (st = check_given({x, adapter_ids, a, b, out}, err)) ||
        (st = lora_apart(x, x_dtype, adapter_ids, a, b, w_dtype, scales, m, n, k, rank, adapters, base, out, out_dtype, h_out, err)))
        return st;
    return guarded(err, [&]() -> nh_status {
        std::vector<float> h(rank);
        for (size_t i = 0; i < m; ++i) {
            const int32_t l = adapter_ids[i];
            const bool has = l >= 0 && (size_t)l < adapters;
            const double s = has && scales ? (double)scales[l] : 1.0;
            for (size_t r = 0; r < rank; ++r) {
                double v = 0.0;
                for (size_t c = 0; has && c < k; ++c)
                    v += (double)load_f32(x, i * k + c, x_dtype) * (double)load_f32(a, ((size_t)l * rank + r) * k + c, w_dtype);
                h[r] = (float)v;
                if (h_out) h_out[i * rank + r] = h[r];
            }
            for (size_t c = 0; c < n; ++c) {
                double v = 0.0;
                for (size_t r = 0; has && r < rank; ++r)
                    v += (double)h[r] * (double)load_f32(b, ((size_t)l * n + c) * rank + r, w_dtype);
                const double y = base ? (double)load_f32(base, i * n + c, out_dtype) : 0.0;
                store_f32(out, i * n + c, (float)(has ? y + s * v : y), out_dtype);
            }
        }
        return NH_OK;
    });
}

nh_status nh_linear_lora_backward_host(const void* x, nh_dtype x_dtype, const int32_t* adapter_ids, const void* a,
                                       const void* b, nh_dtype w_dtype, const float* scales, const float* h,
                                       const void* dout, nh_dtype dout_dtype, size_t m, size_t n, size_t k, size_t rank,
                                       size_t adapters, const void* dx_base, void* dx, float* da, float* db,
                                       int accumulate, nh_error* err) {
    clear_error(err);
    nh_status st;
    if ((st = check_lora(m, n, k, rank, adapters, {x_dtype, w_dtype, dout_dtype}, err)) ||
        (st = check_given({adapter_ids, dout}, err)))
        return st;
    if (!dx && !da && !db) return set_error(err, NH_INVALID_PARAMS, "null operand");
    const bool again = db && !h;
    if (((da || again) && (st = check_given({x}, err))) || ((dx || again) && (st = check_given({a}, err))) ||
        ((dx || da) && (st = check_given({b}, err))) ||
        (st = lora_backward_apart(x, x_dtype, adapter_ids, a, b, w_dtype, scales, h, dout, dout_dtype, m, n, k, rank, adapters,
                                  dx_base, dx, da, db, err)))
        return st;
    return guarded(err, [&]() -> nh_status {
        std::vector<double> ga(da ? rank * k : 0), gb(db ? rank * n : 0);
        std::vector<float> dh(rank), low(rank);
        for (size_t i = 0; dx && i < m; ++i)  // rows without an adapter
            if (adapter_ids[i] < 0 || (size_t)adapter_ids[i] >= adapters)
                for (size_t c = 0; c < k; ++c)
                    store_f32(dx, i * k + c, dx_base ? load_f32(dx_base, i * k + c, x_dtype) : 0.0f, x_dtype);
        for (size_t l = 0; l < adapters; ++l) {
            std::fill(ga.begin(), ga.end(), 0.0);
            std::fill(gb.begin(), gb.end(), 0.0);
            const double s = scales ? (double)scales[l] : 1.0;
            for (size_t i = 0; i < m; ++i) {
                if (adapter_ids[i] < 0 || (size_t)adapter_ids[i] != l) continue;
                for (size_t r = 0; (dx || da) && r < rank; ++r) {
                    double v = 0.0;
                    for (size_t c = 0; c < n; ++c)
                        v += (double)load_f32(dout, i * n + c, dout_dtype) * (double)load_f32(b, (l * n + c) * rank + r, w_dtype);
                    dh[r] = (float)(s * v);
                }
                for (size_t r = 0; db && r < rank; ++r) {
                    double v = h ? (double)h[i * rank + r] : 0.0;
                    for (size_t c = 0; !h && c < k; ++c)
                        v += (double)load_f32(x, i * k + c, x_dtype) * (double)load_f32(a, (l * rank + r) * k + c, w_dtype);
                    low[r] = (float)v;
                }
                for (size_t c = 0; dx && c < k; ++c) {
                    double v = dx_base ? (double)load_f32(dx_base, i * k + c, x_dtype) : 0.0;
                    for (size_t r = 0; r < rank; ++r) v += (double)dh[r] * (double)load_f32(a, (l * rank + r) * k + c, w_dtype);
                    store_f32(dx, i * k + c, (float)v, x_dtype);
                }
                for (size_t r = 0; da && r < rank; ++r)
                    for (size_t c = 0; c < k; ++c) ga[r * k + c] += (double)dh[r] * (double)load_f32(x, i * k + c, x_dtype);
                for (size_t c = 0; db && c < n; ++c)
                    for (size_t r = 0; r < rank; ++r)
                        gb[c * rank + r] += s * (double)load_f32(dout, i * n + c, dout_dtype) * (double)low[r];
            }
            for (size_t i = 0; i < ga.size(); ++i)
                da[l * rank * k + i] = (float)(accumulate ? (double)da[l * rank * k + i] + ga[i] : ga[i]);
            for (size_t i = 0; i < gb.size(); ++i)
                db[l * rank * n + i] = (float)(accumulate ? (double)db[l * rank * n + i] + gb[i] : gb[i]);
        }
        return NH_OK;
    });
}

}  // extern "C"
