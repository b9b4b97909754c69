// Host twins of the MXFP4 operators and of the router's balance loss.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <exception>
#include <new>
#include <vector>

#include "../kernels/mx_numerics.h"
#include "../runtime/nh_runtime.h"

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

nh_status find_nonfinite(const void* x, nh_dtype d, size_t n, const char* what, nh_error* err) {
    for (size_t i = 0; i < n; ++i) {
        const float v = load_f32(x, i, d);
        if (std::isfinite(v)) continue;
        if (err) {
            err->argument = what;
            err->index = i;
            err->value = v;
        }
        return set_error(err, NH_NON_FINITE_INPUT, "non-finite %s value %g at index %zu", what, (double)v, i);
    }
    return NH_OK;
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

// One block of `count` values: its scale byte, and their codes.
uint32_t quantize_block(const float* v, size_t count, uint8_t* codes) {
    uint32_t amax = 0;
    for (size_t i = 0; i < count; ++i) amax = std::max(amax, f32_bits(v[i]) & 0x7fffffffu);
    const uint32_t e = mx_scale_byte(amax);
    for (size_t i = 0; i < count; ++i) codes[i] = e == kMxNan ? 0 : (uint8_t)mx_code(v[i], e);
    return e;
}

// A row as the values it is quantized to.
void requantize_row(const void* x, nh_dtype d, size_t row, size_t cols, float* out) {
    float v[kMxBlock];
    uint8_t c[kMxBlock];
    for (size_t b = 0; b < cols; b += kMxBlock) {
        const size_t n = std::min<size_t>(kMxBlock, cols - b);
        for (size_t i = 0; i < n; ++i) v[i] = load_f32(x, row * cols + b + i, d);
        const uint32_t e = quantize_block(v, n, c);
        for (size_t i = 0; i < n; ++i) out[b + i] = mx_value(c[i], e);
    }
}

// Row n of tiled weights as values.
void tiled_row(const uint8_t* w, size_t n, size_t k, float* out) {
    const uint8_t* region = w + n / 16 * mx_region_bytes(k);
    const uint8_t* scales = region + mx_k_tiles(k) * 1024;
    for (size_t i = 0; i < k; ++i) {
        const size_t kt = i / 128, lane = 16 * (i % 128 / 32) + n % 16;
        const uint32_t byte = region[kt * 1024 + lane * 16 + i % 32 / 2];
        out[i] = mx_value((byte >> (4 * (i & 1))) & 15, scales[kt / 4 * 256 + lane * 4 + kt % 4]);
    }
}

float dot(const float* a, const float* b, size_t k, const float* bias, size_t n) {
    double s = 0.0;
    for (size_t i = 0; i < k; ++i) s += (double)a[i] * (double)b[i];
    const float y = (float)s;
    return bias ? y + bias[n] : y;
}

}  // namespace

extern "C" {

nh_status nh_quantize_rows_mxfp4_host(const void* x, nh_dtype dtype, size_t rows, size_t cols, uint8_t* codes,
                                      uint8_t* scales, nh_error* err) {
    clear_error(err);
    nh_status st = check_dtype(dtype, err);
    size_t n;
    if (st) return st;
    if (!mul_ok(rows, cols, &n)) return set_error(err, NH_INVALID_SHAPE, "rows * cols overflows");
    if (n != 0 && (st = check_given({x, codes, scales}, err))) return st;
    if ((st = find_nonfinite(x, dtype, n, "input", err))) return st;
    float v[kMxBlock];
    uint8_t c[kMxBlock];
    const size_t rc = mx_row_codes(cols), rb = mx_row_blocks(cols);
    for (size_t r = 0; r < rows; ++r)
        for (size_t b = 0; b < rb; ++b) {
            const size_t count = std::min<size_t>(kMxBlock, cols - b * kMxBlock);
            for (size_t i = 0; i < count; ++i) v[i] = load_f32(x, r * cols + b * kMxBlock + i, dtype);
            scales[r * rb + b] = (uint8_t)quantize_block(v, count, c);
            for (size_t i = 0; i < count; i += 2)
                codes[r * rc + b * (kMxBlock / 2) + i / 2] = (uint8_t)(c[i] | (i + 1 < count ? c[i + 1] << 4 : 0));
        }
    return NH_OK;
}

nh_status nh_dequantize_mxfp4_host(const uint8_t* codes, const uint8_t* scales, size_t rows, size_t cols, void* out,
                                   nh_dtype out_dtype, nh_error* err) {
    clear_error(err);
    nh_status st = check_dtype(out_dtype, err);
    size_t n;
    if (st) return st;
    if (!mul_ok(rows, cols, &n)) return set_error(err, NH_INVALID_SHAPE, "rows * cols overflows");
    if (n != 0 && (st = check_given({codes, scales, out}, err))) return st;
    const size_t rc = mx_row_codes(cols), rb = mx_row_blocks(cols);
    for (size_t r = 0; r < rows; ++r)
        for (size_t c = 0; c < cols; ++c)
            store_f32(out, r * cols + c, mx_value((codes[r * rc + c / 2] >> (4 * (c & 1))) & 15, scales[r * rb + c / kMxBlock]),
                      out_dtype);
    return NH_OK;
}

nh_status nh_tile_weights_mxfp4_host(const uint8_t* codes, const uint8_t* scales, size_t n, size_t k, uint8_t* tiled,
                                     size_t tiled_len, nh_error* err) {
    clear_error(err);
    const size_t need = nh_tiled_mxfp4_weights_bytes(n, k);
    if (need == 0) return set_error(err, NH_INVALID_SHAPE, "invalid weight shape n=%zu k=%zu", n, k);
    if (tiled_len != need) return mismatch(err, "tiled", need, tiled_len);
    if (nh_status st = check_given({codes, scales, tiled}, err)) return st;
    std::memset(tiled, 0, need);
    const size_t rc = mx_row_codes(k), rb = mx_row_blocks(k);
    for (size_t r = 0; r < n; ++r) {
        uint8_t* region = tiled + r / 16 * mx_region_bytes(k);
        for (size_t b = 0; b < rb; ++b) {
            const size_t kt = b / 4, lane = 16 * (b % 4) + r % 16;
            for (size_t i = 0; i < kMxBlock && b * kMxBlock + i < k; ++i)
                region[kt * 1024 + lane * 16 + i / 2] |=
                    (uint8_t)(((codes[r * rc + b * (kMxBlock / 2) + i / 2] >> (4 * (i & 1))) & 15) << (4 * (i & 1)));
            region[mx_k_tiles(k) * 1024 + kt / 4 * 256 + lane * 4 + kt % 4] = scales[r * rb + b];
        }
    }
    return NH_OK;
}

nh_status nh_linear_mxfp4_host(const void* x, nh_dtype x_dtype, const uint8_t* w, const float* bias, size_t m, size_t n,
                               size_t k, void* out, nh_dtype out_dtype, nh_error* err) {
    clear_error(err);
    if (n == 0 || k == 0) return set_error(err, NH_INVALID_SHAPE, "invalid linear shape k=%zu n=%zu", k, n);
    if (m == 0) return set_error(err, NH_INVALID_ROW_COUNT, "row_count must be non-zero, got 0");
    nh_status st;
    if ((st = check_dtype(x_dtype, err)) || (st = check_dtype(out_dtype, err))) return st;
    size_t mk, mn;
    if (!mul_ok(m, k, &mk) || !mul_ok(m, n, &mn) || nh_tiled_mxfp4_weights_bytes(n, k) == 0)
        return set_error(err, NH_INVALID_SHAPE, "linear shape m=%zu n=%zu k=%zu overflows", m, n, k);
    if ((st = check_given({x, w, out}, err))) return st;
    if ((st = find_nonfinite(x, x_dtype, mk, "input", err))) return st;
    return guarded(err, [&]() -> nh_status {
        std::vector<float> xv(mk), row(k);
        for (size_t i = 0; i < m; ++i) requantize_row(x, x_dtype, i, k, xv.data() + i * k);
        for (size_t j = 0; j < n; ++j) {
            tiled_row(w, j, k, row.data());
            for (size_t i = 0; i < m; ++i)
                store_f32(out, i * n + j, dot(xv.data() + i * k, row.data(), k, bias, j), out_dtype);
        }
        return NH_OK;
    });
}

nh_status nh_moe_forward_mxfp4_host(const void* x, nh_dtype x_dtype, const float* logits, size_t tokens, size_t hidden,
                                    size_t inter, size_t experts, size_t top_k, int renormalize, float scaling,
                                    const uint8_t* w_up, const uint8_t* w_down, const nh_moe_biases* biases,
                                    const float* shared, void* out, nh_dtype out_dtype, nh_error* err) {
    clear_error(err);
    if (tokens == 0) return set_error(err, NH_INVALID_ROW_COUNT, "row_count must be non-zero, got 0");
    size_t routes, n;
    if (hidden == 0 || inter == 0 || experts == 0 || top_k == 0 || top_k > experts || !mul_ok(tokens, top_k, &routes) ||
        routes >= (1ull << 31) || !mul_ok(tokens, hidden, &n) || !mul_ok(tokens, experts, &n) || !mul_ok(routes, hidden, &n) ||
        !mul_ok(routes, inter, &n) || !nh_tiled_mxfp4_weights_bytes(inter, hidden) || !nh_tiled_mxfp4_weights_bytes(hidden, inter))
        return set_error(err, NH_INVALID_SHAPE, "invalid MoE shape");
    if (biases && (biases->shared_up || biases->shared_down))
        return set_error(err, NH_INVALID_PARAMS, "shared expert biases given without a shared expert");
    nh_status st;
    if ((st = check_dtype(x_dtype, err)) || (st = check_dtype(out_dtype, err))) return st;
    if ((st = check_given({x, logits, w_up, w_down, out}, err))) return st;
    if ((st = find_nonfinite(x, x_dtype, tokens * hidden, "input", err))) return st;
    return guarded(err, [&]() -> nh_status {
        std::vector<int32_t> idx(routes), offsets(experts + 1), perm(routes), pos(routes);
        std::vector<float> wts(routes), xv(tokens * hidden), h(routes * inter), hq(inter), d(routes * hidden), row;
        if ((st = nh_moe_route_sigmoid_topk_host(logits, tokens * experts, tokens, experts, top_k, renormalize, scaling,
                                                 idx.data(), routes, wts.data(), routes, err)))
            return st;
        if ((st = nh_moe_permute_host(idx.data(), tokens, top_k, experts, offsets.data(), perm.data(), pos.data(), err)))
            return st;
        for (size_t t = 0; t < tokens; ++t) requantize_row(x, x_dtype, t, hidden, xv.data() + t * hidden);
        const float *b_up = biases ? biases->up : nullptr, *b_down = biases ? biases->down : nullptr;
        row.resize(std::max(hidden, inter));
        for (size_t e = 0; e < experts; ++e) {
            const size_t s0 = (size_t)offsets[e], s1 = (size_t)offsets[e + 1];
            if (s0 == s1) continue;
            for (size_t j = 0; j < inter; ++j) {
                tiled_row(w_up + e * nh_tiled_mxfp4_weights_bytes(inter, hidden), j, hidden, row.data());
                for (size_t s = s0; s < s1; ++s) {
                    // a NaN (of a weight's block with no value) stays one, as on the device
                    const float y = dot(xv.data() + (size_t)perm[s] / top_k * hidden, row.data(), hidden,
                                        b_up ? b_up + e * inter : nullptr, j);
                    h[s * inter + j] = y != y ? y : relu2(y);
                }
            }
        }
        if ((st = find_nonfinite(h.data(), NH_F32, h.size(), "intermediate", err))) return st;
        for (size_t s = 0; s < routes; ++s) {
            requantize_row(h.data(), NH_F32, s, inter, hq.data());
            std::copy(hq.begin(), hq.end(), h.begin() + s * inter);
        }
        for (size_t e = 0; e < experts; ++e) {
            const size_t s0 = (size_t)offsets[e], s1 = (size_t)offsets[e + 1];
            for (size_t j = 0; s0 < s1 && j < hidden; ++j) {
                tiled_row(w_down + e * nh_tiled_mxfp4_weights_bytes(hidden, inter), j, inter, row.data());
                for (size_t s = s0; s < s1; ++s)
                    d[s * hidden + j] =
                        dot(h.data() + s * inter, row.data(), inter, b_down ? b_down + e * hidden : nullptr, j);
            }
        }
        return nh_moe_combine_shared_host(d.data(), pos.data(), wts.data(), shared, tokens, top_k, hidden, out, out_dtype, err);
    });
}

}  // extern "C"

namespace {

nh_status check_balance(size_t sequences, const int32_t* off, size_t tokens, size_t experts, size_t top_k,
                        float coefficient, nh_error* err) {
    size_t n;
    if (experts == 0 || top_k == 0 || sequences == 0 || (!off && sequences != 1) || !mul_ok(tokens, experts, &n) ||
        !mul_ok(tokens, top_k, &n) || !mul_ok(sequences, experts, &n))
        return set_error(err, NH_INVALID_SHAPE, "invalid balance shape sequences=%zu experts=%zu top_k=%zu", sequences,
                         experts, top_k);
    if (!std::isfinite(coefficient)) return set_error(err, NH_INVALID_PARAMS, "coefficient must be finite");
    return NH_OK;
}

// Tokens [lo, hi) of sequence s, offsets out of range or order as on the device.
void bounds(const int32_t* off, size_t s, size_t tokens, size_t* lo, size_t* hi) {
    const int64_t t = (int64_t)tokens;
    const int64_t l = off ? std::min(std::max<int64_t>(off[s], 0), t) : 0;
    *lo = (size_t)l;
    *hi = (size_t)(off ? std::min(std::max<int64_t>(off[s + 1], l), t) : t);
}

// The row's probabilities, and d of each.
void probabilities(const float* z, size_t experts, int softmax, double* p, double* slope) {
    double m = -INFINITY, sum = 0.0;
    for (size_t e = 0; e < experts; ++e) m = std::max(m, (double)z[e]);  // skips a NaN
    const bool none = m == -INFINITY;
    if (none) m = 0.0;
    if (!softmax) m = std::min(m, 0.0);
    for (size_t e = 0; e < experts; ++e) {
        const double v = z[e];
        if (softmax) {
            p[e] = std::exp(v - m);
            slope[e] = 1.0;
        } else {
            const double d = 1.0 + std::exp(-std::fabs(v));
            p[e] = v != v ? v : std::exp(std::min(v, 0.0) - m) / d;
            slope[e] = std::exp(-std::max(v, 0.0)) / d;
        }
        sum += p[e];
    }
    for (size_t e = 0; e < experts; ++e) p[e] = none && sum == sum ? 0.0 : p[e] / sum;
}

}  // namespace

extern "C" {

nh_status nh_moe_balance_loss_host(const float* logits, const int32_t* indices, const int32_t* seq_offsets,
                                   size_t sequences, size_t tokens, size_t experts, size_t top_k, int softmax,
                                   float coefficient, int32_t* counts, float* loss, nh_error* err) {
    clear_error(err);
    nh_status st = check_balance(sequences, seq_offsets, tokens, experts, top_k, coefficient, err);
    if (st) return st;
    if ((st = check_given({counts, loss}, err))) return st;
    if (tokens != 0 && (st = check_given({logits, indices}, err))) return st;
    return guarded(err, [&]() -> nh_status {
        std::vector<double> p(experts), slope(experts), sums(experts);
        double total = 0.0;
        for (size_t s = 0; s < sequences; ++s) {
            size_t lo, hi;
            bounds(seq_offsets, s, tokens, &lo, &hi);
            std::fill(sums.begin(), sums.end(), 0.0);
            int32_t* c = counts + s * experts;
            std::fill(c, c + experts, 0);
            for (size_t t = lo; t < hi; ++t) {
                probabilities(logits + t * experts, experts, softmax, p.data(), slope.data());
                for (size_t e = 0; e < experts; ++e) sums[e] += p[e];
                for (size_t j = 0; j < top_k; ++j) {
                    const int32_t e = indices[t * top_k + j];
                    if (e >= 0 && (size_t)e < experts) ++c[e];
                }
            }
            double dot = 0.0;
            const double n = (double)(hi - lo);
            for (size_t e = 0; e < experts; ++e) dot += (double)c[e] * sums[e];
            if (hi > lo) total += (double)coefficient / (double)sequences * dot * (double)experts / ((double)top_k * n * n);
        }
        *loss = (float)total;
        return NH_OK;
    });
}

nh_status nh_moe_balance_loss_backward_host(const float* logits, const int32_t* counts, const int32_t* seq_offsets,
                                            size_t sequences, size_t tokens, size_t experts, size_t top_k, int softmax,
                                            float coefficient, const float* dloss, float* dlogits, nh_error* err) {
    clear_error(err);
    nh_status st = check_balance(sequences, seq_offsets, tokens, experts, top_k, coefficient, err);
    if (st) return st;
    if (tokens != 0 && (st = check_given({logits, counts, dloss, dlogits}, err))) return st;
    std::fill(dlogits, dlogits + tokens * experts, 0.0f);
    return guarded(err, [&]() -> nh_status {
        std::vector<double> p(experts), slope(experts);
        for (size_t s = 0; s < sequences; ++s) {
            size_t lo, hi;
            bounds(seq_offsets, s, tokens, &lo, &hi);
            const double n = (double)(hi - lo), per = (double)experts / ((double)top_k * n);
            for (size_t t = lo; t < hi; ++t) {
                probabilities(logits + t * experts, experts, softmax, p.data(), slope.data());
                double fp = 0.0;
                for (size_t e = 0; e < experts; ++e) fp += (double)counts[s * experts + e] * per * p[e];
                for (size_t e = 0; e < experts; ++e)
                    dlogits[t * experts + e] = (float)((double)*dloss * (double)coefficient / ((double)sequences * n) * p[e] *
                                                       ((double)counts[s * experts + e] * per - fp) * slope[e]);
            }
        }
        return NH_OK;
    });
}

}  // extern "C"
