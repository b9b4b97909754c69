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
#include "nh_device.h"

using namespace nh;

namespace {

constexpr int kBalanceWaves = 16;

// The sequence of chunk b and its tokens [lo, hi); s = -1: there is no such chunk.
__device__ __forceinline__ int balance_bounds(const BalanceArgs& a, int s, int& lo, int& hi) {
    lo = 0;
    hi = a.tokens;
    if (a.seq) {  // offsets out of range or order are taken as the nearest valid ones
        lo = min(max(a.seq[s], 0), a.tokens);
        hi = min(max(a.seq[s + 1], lo), a.tokens);
    }
    return hi - lo;
}

__device__ __forceinline__ int balance_chunk(const BalanceArgs& a, int b, int lane, int& lo, int& hi, int& first) {
    int carry = 0;
    for (int base = 0; base < a.sequences; base += 64) {
        const int s = base + lane;
        int l = 0, h = 0;
        const int n = s < a.sequences ? balance_bounds(a, s, l, h) : 0;
        const int mine = (n + a.chunk - 1) / a.chunk;
        int incl = mine;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int t = __shfl_up(incl, off, kWave);
            if (lane >= off) incl += t;
        }
        const uint64_t past = __ballot(carry + incl > b);
        if (past) {
            const int at = __ffsll((unsigned long long)past) - 1;
            const int j = b - (carry + __builtin_amdgcn_readlane(incl - mine, at));  // chunk of the sequence
            first = __builtin_amdgcn_readlane(l, at);
            lo = first + j * a.chunk;
            hi = min(lo + a.chunk, __builtin_amdgcn_readlane(h, at));
            return base + at;
        }
        carry += __builtin_amdgcn_readlane(incl, 63);
    }
    return -1;
}

__device__ __forceinline__ float group_max(float v, int group) {
    for (int off = group >> 1; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, kWave));
    return v;
}

__device__ __forceinline__ float group_sum(float v, int group) {
    for (int off = group >> 1; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
    return v;
}

// A token's logits: lane j of the group holds experts 4 (j + i group) .. + 3 in
// turn i; experts past E are -inf.
template <int S>
__device__ __forceinline__ void balance_row(const BalanceArgs& a, int64_t token, int j, bool ok, float (&z)[S][4]) {
    const int E = a.experts;
#pragma unroll
    for (int i = 0; i < S; ++i) {
        const int e = 4 * (j + i * a.group);
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

// The row's probabilities in place of its logits; slope: d of each (sigmoid).
template <int S, bool SLOPE>
__device__ __forceinline__ void balance_probabilities(const BalanceArgs& a, float (&z)[S][4], float (&slope)[S][4]) {
    float m = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) m = fmaxf(m, z[i][q]);
    m = group_max(m, a.group);
    const bool none = m == -__builtin_inff();
    if (!a.softmax) m = fminf(m, 0.0f);
    if (none) m = 0.0f;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float v = z[i][q];
            if (a.softmax) {
                z[i][q] = __expf(v - m);
            } else {
                const float d = 1.0f + __expf(-fabsf(v));
                z[i][q] = __expf(fminf(v, 0.0f) - m) / d;
                if constexpr (SLOPE) slope[i][q] = __expf(-fmaxf(v, 0.0f)) / d;
                if (v != v) z[i][q] = v;  // the minimum drops a NaN
            }
            sum += z[i][q];
        }
    sum = group_sum(sum, a.group);
    const float r = none && !(sum != sum) ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) z[i][q] *= r;
}

template <int S>
__device__ __forceinline__ void balance_partial(const BalanceArgs& a, int* lds) {
    const int E = a.experts, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int lo, hi, first;
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.arrived = 0;
    const int s = balance_chunk(a, blockIdx.x, lane, lo, hi, first);
    if (s < 0) return;  // uniform
    int* hist = lds;                    // [E]
    float* psum = (float*)(lds + E);    // [waves][E]
    for (int e = threadIdx.x; e < E; e += blockDim.x) hist[e] = 0;
    __syncthreads();
    const int64_t r1 = (int64_t)hi * a.top_k;
    for (int64_t r = (int64_t)lo * a.top_k + threadIdx.x; r < r1; r += blockDim.x) {
        const int e = a.indices[r];
        if (e >= 0 && e < E) atomicAdd(&hist[e], 1);
    }
    const int rows = 64 / a.group, j = lane & (a.group - 1), row = lane / a.group;
    float acc[S][4];
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[i][q] = 0.0f;
    for (int t0 = lo + wave * rows; t0 < hi; t0 += kBalanceWaves * rows) {
        const bool ok = t0 + row < hi;
        float z[S][4], none[S][4];
        balance_row<S>(a, t0 + row, j, ok, z);
        balance_probabilities<S, false>(a, z, none);
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[i][q] += z[i][q];
    }
    // the wave's rows, then the waves in order
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float v = acc[i][q];
            for (int off = 32; off >= a.group; off >>= 1) v += __shfl_xor(v, off, kWave);
            const int e = 4 * (j + i * a.group) + q;
            if (row == 0 && e < E) psum[wave * E + e] = v;
        }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += blockDim.x) {
        float v = psum[e];
        for (int w = 1; w < kBalanceWaves; ++w) v += psum[w * E + e];
        a.part_p[(int64_t)blockIdx.x * E + e] = v;
        a.part_n[(int64_t)blockIdx.x * E + e] = hist[e];
    }
}

}  // namespace

extern "C" __global__ __launch_bounds__(64 * kBalanceWaves) void nh_moe_balance_partial_kernel(BalanceArgs a) {
    extern __shared__ int balance_lds[];
    if (a.experts <= 256)
        balance_partial<1>(a, balance_lds);
    else
        balance_partial<4>(a, balance_lds);
}

// One workgroup per sequence: its chunks' sums in order, its counts and loss;
// the last workgroup to finish adds the sequences' losses, in order.
extern "C" __global__ __launch_bounds__(1024) void nh_moe_balance_reduce_kernel(BalanceArgs a) {
    extern __shared__ int balance_lds[];
    const int E = a.experts, s = blockIdx.x, lane = threadIdx.x & 63;
    // chunks of the sequences before this one
    int before = 0;
    for (int i = lane; i < s; i += 64) {
        int l, h;
        before += (balance_bounds(a, i, l, h) + a.chunk - 1) / a.chunk;
    }
    for (int off = 32; off > 0; off >>= 1) before += __shfl_xor(before, off, kWave);
    int lo, hi;
    const int n = balance_bounds(a, s, lo, hi);
    const int chunks = min((n + a.chunk - 1) / a.chunk, a.chunks - before);  // offsets that overlap: no more than there are
    // threads by expert and by residue of the chunk
    const int cols = min(E, 1024), parts = 1024 / cols, col = threadIdx.x % cols, part = threadIdx.x / cols;
    double* red = (double*)balance_lds;      // [16]
    float* ps = (float*)(red + 16);          // [parts][cols]
    int* ns = (int*)(ps + 1024);             // [parts][cols]
    float v = 0.0f;
    int c = 0;
    if (part < parts) {
#pragma unroll 8
        for (int i = part; i < chunks; i += parts) {
            v += a.part_p[(int64_t)(before + i) * E + col];
            c += a.part_n[(int64_t)(before + i) * E + col];
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
            p += (double)ps[i * cols + threadIdx.x];
            total += ns[i * cols + threadIdx.x];
        }
        a.counts[(int64_t)s * E + threadIdx.x] = total;
        dot = p * (double)total;
    }
    dot = wave_sum_f64(dot);
    if (lane == 0) red[threadIdx.x >> 6] = dot;
    __syncthreads();
    if (threadIdx.x != 0) return;
    double sum = 0.0;
    for (int w = 0; w < 16; ++w) sum += red[w];
    const double scale = (double)a.coefficient / (double)a.sequences;
    const double mine = n > 0 ? scale * sum * (double)E / ((double)a.top_k * (double)n * (double)n) : 0.0;
    if (a.sequences == 1) {
        a.loss[0] = (float)mine;
        return;
    }
    __hip_atomic_store((uint64_t*)&a.seq_loss[s], f64_bits(mine), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const uint32_t order = __hip_atomic_fetch_add(a.arrived, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    if (order + 1 != (uint32_t)a.sequences) return;
    double total = 0.0;
    for (int i = 0; i < a.sequences; ++i)
        total += f64_from_bits(__hip_atomic_load((uint64_t*)&a.seq_loss[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    a.loss[0] = (float)total;
}

namespace {

template <int S>
__device__ __forceinline__ void balance_backward(const BalanceArgs& a) {
    const int E = a.experts, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int rows = 64 / a.group, j = lane & (a.group - 1), row = lane / a.group;
    const int64_t waves = (int64_t)gridDim.x * (blockDim.x >> 6);
    const float up = a.dloss[0] * a.coefficient / (float)a.sequences;
    int s = -1, lo = 0, hi = 0;  // the group's sequence, its f and scale
    float f[S][4], scale = 0.0f;
    for (int64_t t0 = ((int64_t)blockIdx.x * (blockDim.x >> 6) + wave) * rows; t0 < a.tokens; t0 += waves * rows) {
        const int t = (int)t0 + row;
        const bool ok = t < a.tokens;
        float z[S][4], slope[S][4];
        balance_row<S>(a, t, j, ok, z);
        if (s < 0 || t >= hi) {
            // the first sequence that ends behind t
            int b = 0, e = a.sequences - 1;
            while (b < e) {
                const int m = (b + e) >> 1;
                if (balance_bounds(a, m, lo, hi), hi > t) e = m;
                else b = m + 1;
            }
            s = b;
            const int n = balance_bounds(a, s, lo, hi);
            scale = n > 0 ? up / (float)n : 0.0f;
            const float per = n > 0 ? (float)E / ((float)a.top_k * (float)n) : 0.0f;
#pragma unroll
            for (int i = 0; i < S; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int x = 4 * (j + i * a.group) + q;
                    f[i][q] = x < E ? (float)a.counts[(int64_t)s * E + x] * per : 0.0f;
                }
        }
        balance_probabilities<S, true>(a, z, slope);
        float fp = 0.0f;
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) fp += f[i][q] * z[i][q];
        fp = group_sum(fp, a.group);
        const bool in = t >= lo && t < hi;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const int e = 4 * (j + i * a.group);
            float d[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                d[q] = scale * z[i][q] * (f[i][q] - fp);
                if (!a.softmax) d[q] *= slope[i][q];
                if (!in) d[q] = 0.0f;  // behind the last sequence
            }
            float* at = a.dlogits + (int64_t)t * E + e;
            if (ok && e + 3 < E) {
                __builtin_memcpy(at, d, 16);
            } else if (ok) {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (e + q < E) at[q] = d[q];
            }
        }
    }
}

}  // namespace

extern "C" __global__ __launch_bounds__(256) void nh_moe_balance_backward_kernel(BalanceArgs a) {
    if (a.experts <= 256)
        balance_backward<1>(a);
    else
        balance_backward<4>(a);
}
