// Load balance of the router: routes per expert, the balance loss and its
// gradient with respect to the logits.
//
// For a sequence of n tokens with top_k routes each over E experts:
//   f_e = E / (top_k n) * (its routes to e),   p_te = the router's probability,
//   L_s = 1 / n * sum_t sum_e f_e p_te,        L = c / S * sum_s L_s.
// The counts take no gradient, so
//   dL/dz_te = c / (S n) * p_te (f_e - sum_j f_j p_tj) * d_te,
// d = 1 for p = softmax(z) and d = 1 - sigmoid(z_te) for p = sigmoid(z) / sum
// of the row's sigmoids.  That p is evaluated as u / sum u with
//   u = exp(min(z, 0) - min(max z, 0)) / (1 + exp(-|z|)),
// the sigmoids over a common factor, so that a row of large negative logits
// keeps its ratios.  A row of -inf alone has no probabilities: it adds nothing
// and its gradient is 0.
//
// Bound by the logits' bytes (read once forward, read and written once
// backward) and, for few tokens, by the launches.  `group` lanes share a token,
// four consecutive experts (one 16-byte load) per lane and turn, so a row meets
// in log2(group) lane moves and a wave takes 64 / group rows at once.
// Every sum has a fixed order: results do not change from run to run.
// 131072 x 128: 22.5 us for the loss's partial sums (67 MB, 3.0 TB/s), 6.6 to join
// them, 26 for the gradient (134 MB, 5.2 TB/s); 64 x 128 5.7 and 5.1.
#include "nh_device.h"

using namespace nh;

namespace {

constexpr int kBalanceWaves = 16;

// The tokens [lo, hi) of sequence s, and how many.
__device__ __forceinline__ int balance_bounds(const BalanceArgs& a, int s, int& lo, int& hi) {
    lo = 0;
    hi = a.tokens;
    if (a.seq) {  // offsets out of range or order are taken as the nearest valid ones
        lo = min(max(a.seq[s], 0), a.tokens);
        hi = min(max(a.seq[s + 1], lo), a.tokens);
    }
    return hi - lo;
}

// Sums over the lanes up to this one.
__device__ __forceinline__ int wave_scan_i32(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr 1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);  // row_shr 2
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);  // row_shr 4
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);  // row_shr 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast 15
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast 31
    return v;
}

// Offsets of 64 sequences each that a walk over them has in flight (131072 x 128
// in 1024 sequences, forward and backward: 234 us one at a time through
// LDS-crossbar scans, 117 so).
constexpr int kSequenceLoads = 4;

__device__ __forceinline__ int balance_chunks(const BalanceArgs& a, int n) { return (n + a.chunk - 1) / a.chunk; }

// The sequence of chunk b, its length n and the chunk's tokens [lo, hi); s = -1:
// there is no such chunk.
__device__ __forceinline__ int balance_chunk(const BalanceArgs& a, int b, int lane, int& lo, int& hi, int& n) {
    int carry = 0;
    for (int base = 0; base < a.sequences; base += 64 * kSequenceLoads) {
        int l[kSequenceLoads], h[kSequenceLoads];
#pragma unroll
        for (int i = 0; i < kSequenceLoads; ++i) balance_bounds(a, min(base + 64 * i + lane, a.sequences - 1), l[i], h[i]);
#pragma unroll
        for (int i = 0; i < kSequenceLoads; ++i) {
            if (base + 64 * i >= a.sequences) break;  // uniform
            const int mine = base + 64 * i + lane < a.sequences ? balance_chunks(a, h[i] - l[i]) : 0;
            const int incl = wave_scan_i32(mine);
            const uint64_t past = __ballot(carry + incl > b);
            if (past) {
                const int at = __ffsll((unsigned long long)past) - 1;
                const int j = b - (carry + __builtin_amdgcn_readlane(incl - mine, at));  // chunk of the sequence
                const int first = __builtin_amdgcn_readlane(l[i], at), end = __builtin_amdgcn_readlane(h[i], at);
                lo = first + j * a.chunk;
                hi = min(lo + a.chunk, end);
                n = end - first;
                return base + 64 * i + at;
            }
            carry += __builtin_amdgcn_readlane(incl, 63);
        }
    }
    return -1;
}

// Maximum and sum over the lanes of a token (G consecutive lanes, every one of
// them gets it): lane moves within rows of 16, then swaps of rows and halves.
template <int CTRL>
__device__ __forceinline__ float dpp_move(float v) {
    return f32_from_bits((uint32_t)__builtin_amdgcn_update_dpp((int)f32_bits(v), (int)f32_bits(v), CTRL, 0xf, 0xf, false));
}

template <int G, class Op>
__device__ __forceinline__ float group_reduce(float v, Op op) {
    if constexpr (G >= 2) v = op(v, dpp_move<0xb1>(v));    // quad_perm 1,0,3,2
    if constexpr (G >= 4) v = op(v, dpp_move<0x4e>(v));    // quad_perm 2,3,0,1
    if constexpr (G >= 8) v = op(v, dpp_move<0x141>(v));   // row_half_mirror
    if constexpr (G >= 16) v = op(v, dpp_move<0x140>(v));  // row_mirror
    if constexpr (G >= 32) {
        const auto t = __builtin_amdgcn_permlane16_swap(f32_bits(v), f32_bits(v), false, false);
        v = op(f32_from_bits(t[0]), f32_from_bits(t[1]));
    }
    if constexpr (G >= 64) {
        const auto t = __builtin_amdgcn_permlane32_swap(f32_bits(v), f32_bits(v), false, false);
        v = op(f32_from_bits(t[0]), f32_from_bits(t[1]));
    }
    return v;
}

// A token's logits: lane j of its G holds experts 4 (j + i G) .. + 3 in turn i;
// experts past E, and every one where !ok, are -inf.
template <int G, int S>
__device__ __forceinline__ void balance_row(const BalanceArgs& a, int64_t token, int j, bool ok, float (&z)[S][4]) {
    const int E = a.experts;
#pragma unroll
    for (int i = 0; i < S; ++i) {
        const int e = 4 * (j + i * G);
        const float* at = a.logits + token * E + e;
#pragma unroll
        for (int q = 0; q < 4; ++q) z[i][q] = -__builtin_inff();
        if (ok && e + 3 < E) {
            __builtin_memcpy(z[i], at, 16);
        } else if (ok) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (e + q < E) z[i][q] = at[q];
        }
    }
}

// exp(x), x <= 0 or a NaN: 2^t, t = x log2 e as rounded, times 1 + (x - t ln 2),
// ln 2 in two parts: off by the 2^-23 of v_exp_f32 and a rounding whatever x
// (2^t alone by |x| 2^-24).  v_exp_f32 gives 0 below the normal range.  x stops
// at -128 (2^-184): an infinity's difference would be a NaN.
__device__ __forceinline__ float exp_nonpositive(float x) {
    constexpr float kLn2 = 0x1.62e43p-1f, kLn2Rest = -0x1.05c61p-29f;
    x = __builtin_elementwise_maximum(x, -128.0f);  // a NaN stays one
    const float t = x * 0x1.715476p+0f;
    const float r = __builtin_fmaf(-t, kLn2Rest, __builtin_fmaf(-t, kLn2, x));
    const float p = __builtin_amdgcn_exp2f(t);
    return __builtin_fmaf(p, r, p);
}

// The row's u in place of its logits, returning 1 / sum u (p = u / sum u); slope:
// d of each (sigmoid).  p is off by the rounding of the difference from the row's
// largest logit (2^-24 of it; none in a sigmoid), the 2^-23 of v_exp_f32 and of
// v_rcp_f32, and a few half steps.  An exp of a NaN is one, so is its row.
template <int G, int S, bool SOFTMAX, bool SLOPE>
__device__ __forceinline__ float balance_probabilities(float (&z)[S][4], float (&slope)[S][4]) {
    float m = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) m = fmaxf(m, z[i][q]);
    m = group_reduce<G>(m, [](float x, float y) { return fmaxf(x, y); });
    const bool none = m == -__builtin_inff();
    if (!SOFTMAX) m = fminf(m, 0.0f);
    if (none) m = 0.0f;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float v = z[i][q];
            if constexpr (SOFTMAX) {
                z[i][q] = exp_nonpositive(v - m);
            } else {
                const float t = exp_nonpositive(-fabsf(v)), r = __builtin_amdgcn_rcpf(1.0f + t);
                // exp(min(v, 0) - m): t itself unless the row's sigmoids are all below 1/2
                z[i][q] = r * (m < 0.0f ? exp_nonpositive(v - m) : v >= 0.0f ? 1.0f : t);
                if constexpr (SLOPE) slope[i][q] = r * (v >= 0.0f ? t : 1.0f);
            }
            sum += z[i][q];
        }
    sum = group_reduce<G>(sum, [](float x, float y) { return x + y; });
    return none && !(sum != sum) ? 0.0f : __builtin_amdgcn_rcpf(sum);
}

// Rows that a wave has in flight per lane group: loads and lane moves of one
// row are a chain, and several interleave (131072 x 128, forward and backward:
// 72 us one row at a time through LDS-crossbar moves, 53 so).  One past 256
// experts, where four rows' registers leave few waves.
constexpr int balance_rows(int turns) { return turns == 1 ? 4 : 1; }

template <int G, int S, bool SOFTMAX>
__device__ __forceinline__ void balance_partial(const BalanceArgs& a, int* lds, int lo, int hi) {
    const int E = a.experts, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int* hist = lds;                    // [E]
    float* psum = (float*)(lds + E);    // [waves][E]
    for (int e = threadIdx.x; e < E; e += blockDim.x) hist[e] = 0;
    __syncthreads();
    // the chunk's routes: the first loads go out ahead of the logits, and count behind them
    const int64_t r0 = (int64_t)lo * a.top_k + threadIdx.x, r1 = (int64_t)hi * a.top_k;
    constexpr int kEarly = 4;
    int early[kEarly];
#pragma unroll
    for (int u = 0; u < kEarly; ++u) early[u] = r0 + u * 64 * kBalanceWaves < r1 ? a.indices[r0 + u * 64 * kBalanceWaves] : -1;
    constexpr int rows = 64 / G, kBalanceRows = balance_rows(S);
    const int j = lane & (G - 1), row = lane / G;
    float acc[S][4];
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[i][q] = 0.0f;
    for (int t0 = lo + wave * rows * kBalanceRows; t0 < hi; t0 += kBalanceWaves * rows * kBalanceRows) {
        float z[kBalanceRows][S][4], none[S][4];
#pragma unroll
        for (int u = 0; u < kBalanceRows; ++u) {
            const int t = t0 + u * rows + row;
            balance_row<G, S>(a, t, j, t < hi, z[u]);
        }
#pragma unroll
        for (int u = 0; u < kBalanceRows; ++u) {
            const float r = balance_probabilities<G, S, SOFTMAX, false>(z[u], none);
#pragma unroll
            for (int i = 0; i < S; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) acc[i][q] = __builtin_fmaf(z[u][i][q], r, acc[i][q]);
        }
    }
    auto count = [&](int e) {
        if (e >= 0 && e < E) atomicAdd(&hist[e], 1);
    };
#pragma unroll
    for (int u = 0; u < kEarly; ++u) count(early[u]);
    for (int64_t r = r0 + kEarly * 64 * kBalanceWaves; r < r1; r += 64 * kBalanceWaves) count(a.indices[r]);
    // the wave's rows, then the waves in order
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float v = acc[i][q];
#pragma unroll
            for (int off = 32; off >= G; off >>= 1) v += __shfl_xor(v, off, kWave);
            const int e = 4 * (j + i * G) + q;
            if (row == 0 && e < E) psum[wave * E + e] = v;
        }
    __syncthreads();
}

// A body per lanes a token has (and turns, past 256 experts) and kind of
// probability.  (32768 x 512, sigmoid, forward and backward: 42 and 35 us in four
// turns, half of them of nothing, 36 and 30 in two.)
#define NH_BALANCE_FORMS(call)                                             \
    switch (a.experts <= 256 ? a.group : a.experts <= 512 ? 128 : 256) {   \
        case 1: call(1, 1); break;                                         \
        case 2: call(2, 1); break;                                         \
        case 4: call(4, 1); break;                                         \
        case 8: call(8, 1); break;                                         \
        case 16: call(16, 1); break;                                       \
        case 32: call(32, 1); break;                                       \
        case 64: call(64, 1); break;                                       \
        case 128: call(64, 2); break;                                      \
        default: call(64, 4); break;                                       \
    }

}  // namespace

// One chunk of a sequence's tokens per workgroup; with one chunk in all
// (a.single) the counts and the loss at once.
extern "C" __global__ __launch_bounds__(64 * kBalanceWaves) void nh_moe_balance_partial_kernel(BalanceArgs a) {
    extern __shared__ int balance_lds[];
    const int E = a.experts, lane = threadIdx.x & 63;
    if (blockIdx.x == 0 && threadIdx.x == 0 && !a.single) *a.arrived = 0;
    int lo, hi, n;
    if (a.single) {
        n = balance_bounds(a, 0, lo, hi);
    } else if (balance_chunk(a, blockIdx.x, lane, lo, hi, n) < 0) {
        return;  // uniform
    }
#define NH_CALL(G, S)                                               \
    if (a.softmax) balance_partial<G, S, true>(a, balance_lds, lo, hi); \
    else balance_partial<G, S, false>(a, balance_lds, lo, hi)
    NH_BALANCE_FORMS(NH_CALL)
#undef NH_CALL
    const int* hist = balance_lds;
    const float* psum = (const float*)(balance_lds + E);
    double dot = 0.0;
    for (int e = threadIdx.x; e < E; e += blockDim.x) {
        float v = psum[e];
        for (int w = 1; w < kBalanceWaves; ++w) v += psum[w * E + e];
        if (a.single) {
            a.counts[e] = hist[e];
            dot += (double)v * (double)hist[e];
        } else {
            a.part_p[(int64_t)blockIdx.x * E + e] = v;
            a.part_n[(int64_t)blockIdx.x * E + e] = hist[e];
        }
    }
    if (!a.single) return;
    dot = wave_sum_f64(dot);
    __syncthreads();  // the partial sums are read
    double* red = (double*)(balance_lds + (E & ~1));
    if (lane == 0) red[threadIdx.x >> 6] = dot;
    __syncthreads();
    if (threadIdx.x != 0) return;
    double sum = 0.0;
    for (int w = 0; w < kBalanceWaves; ++w) sum += red[w];
    const double length = (double)n;
    a.loss[0] = n > 0 ? (float)((double)a.coefficient * sum * (double)E / ((double)a.top_k * length * length)) : 0.0f;
}

// One workgroup per sequence: its chunks' sums in order, its counts and loss;
// the last workgroup to finish adds the sequences' losses, in order.
extern "C" __global__ __launch_bounds__(1024) void nh_moe_balance_reduce_kernel(BalanceArgs a) {
    extern __shared__ int balance_lds[];
    const int E = a.experts, s = blockIdx.x, lane = threadIdx.x & 63;
    // chunks of the sequences before this one
    int before = 0, lo, hi;
    const int n = balance_bounds(a, s, lo, hi);
    for (int base = 0; base < s; base += 64 * kSequenceLoads) {
        int l, h, len[kSequenceLoads];
#pragma unroll
        for (int i = 0; i < kSequenceLoads; ++i) len[i] = balance_bounds(a, min(base + 64 * i + lane, s), l, h);
#pragma unroll
        for (int i = 0; i < kSequenceLoads; ++i) before += base + 64 * i + lane < s ? balance_chunks(a, len[i]) : 0;
    }
    before = __builtin_amdgcn_readlane(wave_scan_i32(before), 63);
    const int chunks = min(balance_chunks(a, n), a.chunks - before);  // offsets that overlap: no more than there are
    // threads by expert and by residue of the chunk
    const int cols = min(E, 1024), parts = 1024 / cols, col = threadIdx.x % cols, part = threadIdx.x / cols;
    double* red = (double*)balance_lds;      // [16]
    double* ps = red + 16;                   // [parts][cols]
    int* ns = (int*)(ps + 1024);             // [parts][cols]
    double v = 0.0;                          // a long sequence has 257 chunks, past 512 experts all of them in one thread
    int c = 0;
    if (part < parts) {
        constexpr int kAhead = 16;  // loads in flight; past the chunks the last one's, unused
        for (int i0 = part; i0 < chunks; i0 += parts * kAhead) {
            float pv[kAhead];
            int pn[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int64_t at = (int64_t)(before + min(i0 + u * parts, chunks - 1)) * E + col;
                pv[u] = a.part_p[at];
                pn[u] = a.part_n[at];
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                v += i0 + u * parts < chunks ? (double)pv[u] : 0.0;
                c += i0 + u * parts < chunks ? pn[u] : 0;
            }
        }
        ps[part * cols + col] = v;
        ns[part * cols + col] = c;
    }
    __syncthreads();
    double dot = 0.0;
    if ((int)threadIdx.x < E) {
        double p = 0.0;
        int total = 0;
        for (int i = 0; i < parts; ++i) {
            p += ps[i * cols + threadIdx.x];
            total += ns[i * cols + threadIdx.x];
        }
        a.counts[(int64_t)s * E + threadIdx.x] = total;
        dot = p * (double)total;
    }
    dot = wave_sum_f64(dot);
    if (lane == 0) red[threadIdx.x >> 6] = dot;
    __syncthreads();
    if (threadIdx.x >= 64) return;
    double sum = 0.0;
#pragma unroll
    for (int w = 0; w < 16; ++w) sum += red[w];
    const double scale = (double)a.coefficient / (double)a.sequences;
    const double mine = n > 0 ? scale * sum * (double)E / ((double)a.top_k * (double)n * (double)n) : 0.0;
    if (a.sequences == 1) {
        if (lane == 0) a.loss[0] = (float)mine;
        return;
    }
    uint32_t order = 0;
    if (lane == 0) {
        __hip_atomic_store((uint64_t*)&a.seq_loss[s], f64_bits(mine), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        order = __hip_atomic_fetch_add(a.arrived, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    }
    if ((uint32_t)__builtin_amdgcn_readfirstlane((int)order) + 1 != (uint32_t)a.sequences) return;
    double total = 0.0;
    for (int i = lane; i < a.sequences; i += 64)
        total += f64_from_bits(__hip_atomic_load((uint64_t*)&a.seq_loss[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    total = wave_sum_f64(total);
    if (lane == 0) a.loss[0] = (float)total;
}

namespace {

template <int G, int S, bool SOFTMAX>
__device__ __forceinline__ void balance_backward(const BalanceArgs& a, int s, int lo, int hi, int n) {
    const int E = a.experts, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    constexpr int rows = 64 / G, kBalanceRows = balance_rows(S);
    const int j = lane & (G - 1), row = lane / G;
    // f and the gradient's scale, of the sequence
    const float scale = a.dloss[0] * a.coefficient / ((float)a.sequences * (float)n);
    const float per = (float)E / ((float)a.top_k * (float)n);
    float f[S][4];
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int e = 4 * (j + i * G) + q;
            f[i][q] = e < E ? (float)a.counts[(int64_t)s * E + e] * per : 0.0f;
        }
    for (int t0 = lo + wave * rows * kBalanceRows; t0 < hi; t0 += waves * rows * kBalanceRows) {
        float z[kBalanceRows][S][4], slope[kBalanceRows][S][4], fp[kBalanceRows];
#pragma unroll
        for (int u = 0; u < kBalanceRows; ++u) {
            const int t = t0 + u * rows + row;
            balance_row<G, S>(a, t, j, t < hi, z[u]);
        }
#pragma unroll
        for (int u = 0; u < kBalanceRows; ++u) {
            const float r = balance_probabilities<G, S, SOFTMAX, true>(z[u], slope[u]);
#pragma unroll
            for (int i = 0; i < S; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) z[u][i][q] *= r;
        }
#pragma unroll
        for (int u = 0; u < kBalanceRows; ++u) {
            fp[u] = 0.0f;
#pragma unroll
            for (int i = 0; i < S; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) fp[u] += f[i][q] * z[u][i][q];
            fp[u] = group_reduce<G>(fp[u], [](float x, float y) { return x + y; });
        }
#pragma unroll
        for (int u = 0; u < kBalanceRows; ++u) {
            const int t = t0 + u * rows + row;
#pragma unroll
            for (int i = 0; i < S; ++i) {
                const int e = 4 * (j + i * G);
                float d[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    d[q] = scale * z[u][i][q] * (f[i][q] - fp[u]);
                    if constexpr (!SOFTMAX) d[q] *= slope[u][i][q];
                }
                float* at = a.dlogits + (int64_t)t * E + e;
                if (t < hi && e + 3 < E) {
                    __builtin_memcpy(at, d, 16);
                } else if (t < hi) {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (e + q < E) at[q] = d[q];
                }
            }
        }
    }
}

}  // namespace

// One chunk of a sequence's tokens per workgroup; the last a.padding workgroups
// clear the rows before the first sequence and behind the last.
extern "C" __global__ __launch_bounds__(256, 4) void nh_moe_balance_backward_kernel(BalanceArgs a) {
    int lo, hi, n;
    if ((int)blockIdx.x >= a.chunks) {
        balance_bounds(a, 0, lo, n);
        balance_bounds(a, a.sequences - 1, n, hi);
        const int64_t head = (int64_t)lo * a.experts, tail = (int64_t)hi * a.experts, end = (int64_t)a.tokens * a.experts;
        const int64_t step = (int64_t)a.padding * blockDim.x;
        const int64_t at = (int64_t)(blockIdx.x - a.chunks) * blockDim.x + threadIdx.x;
        for (int64_t i = at; i < head; i += step) a.dlogits[i] = 0.0f;
        for (int64_t i = tail + at; i < end; i += step) a.dlogits[i] = 0.0f;
        return;
    }
    const int s = balance_chunk(a, blockIdx.x, threadIdx.x & 63, lo, hi, n);
    if (s < 0) return;  // uniform
#define NH_CALL(G, S)                                               \
    if (a.softmax) balance_backward<G, S, true>(a, s, lo, hi, n); \
    else balance_backward<G, S, false>(a, s, lo, hi, n)
    NH_BALANCE_FORMS(NH_CALL)
#undef NH_CALL
}
