// Rows of tokens to the slots of their routes and back, with the routes' weights,
// and the gradients of both.
//
// Route (t, j) has slot s = pos[t k + j] (nh_moe_permute: sorted by expert).
//   scatter: rows[s] = w_tj v_t            dispatch (v = x), backward of the combine (v = dout)
//            dw_tj   = <rows_in[s], v_t>   the combine's weights
//   gather:  out_t   = (shared_t) + sum_j w_tj rows[s]   combine, backward of the dispatch
//            dw_tj   = <rows[s], dot_t>    the dispatch's weights
// A route whose slot is outside [0, slots) takes no part: no row, nothing joined,
// dw = 0.  Slots that no route names are left as they were.
//
// Bound by the rows' bytes: each value of a row is read or written once, each of
// a token once.  One workgroup per token, so that pos and the weights are
// uniform and a weight's gradient is one sum of the workgroup; eight consecutive
// values per thread and turn, as many threads as take the row in the fewest turns.
// Sums run in f32, over j in route order; results do not change from run to run.
#include "nh_device.h"

using namespace nh;

namespace {

constexpr int kRowRoutes = 8;  // routes in flight

// Eight values of a row from column c on, `n` of them there (0: none is read).
template <int DT>
__device__ __forceinline__ void row_load8(const void* p, int64_t at, int n, float (&v)[8]) {
    if constexpr (DT == DT_BF16) {
        const uint16_t* q = (const uint16_t*)p + at;
        if (n >= 8) {
            v4i x;
            __builtin_memcpy(&x, q, 16);
            unpack_bf16x8(x, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = i < n ? bf16_to_f32(q[i]) : 0.0f;
        }
    } else {
        const float* q = (const float*)p + at;
        if (n >= 8) {
            __builtin_memcpy(v, q, 32);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = i < n ? q[i] : 0.0f;
        }
    }
}

template <int DT>
__device__ __forceinline__ void row_store8(void* p, int64_t at, int n, const float (&v)[8]) {
    if constexpr (DT == DT_BF16) {
        uint16_t* q = (uint16_t*)p + at;
        if (n >= 8) {
            const uint32_t x[4] = {f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3]), f32x2_to_bf16x2(v[4], v[5]),
                                   f32x2_to_bf16x2(v[6], v[7])};
            __builtin_memcpy(q, x, 16);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n) q[i] = f32_to_bf16(v[i]);
        }
    } else {
        float* q = (float*)p + at;
        if (n >= 8) {
            __builtin_memcpy(q, v, 32);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n) q[i] = v[i];
        }
    }
}

// The routes j0 .. of token t: their slots (-1: none) and weights.
__device__ __forceinline__ void row_routes(const MoeRowsArgs& a, int64_t t, int j0, int (&slot)[kRowRoutes],
                                           float (&w)[kRowRoutes]) {
#pragma unroll
    for (int j = 0; j < kRowRoutes; ++j) {
        slot[j] = -1;
        w[j] = 1.0f;
        if (j0 + j >= a.top_k) continue;
        const int s = a.pos[t * a.top_k + j0 + j];
        if (s >= 0 && s < a.slots) slot[j] = s;
        if (a.weights) w[j] = a.weights[t * a.top_k + j0 + j];
    }
}

// The workgroup's sums of d, one per route, to dweights.
__device__ __forceinline__ void row_dweights(const MoeRowsArgs& a, int64_t t, int j0, const float (&d)[kRowRoutes],
                                             float (&red)[16][kRowRoutes]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
    for (int j = 0; j < kRowRoutes; ++j) {
        float v = d[j];
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
        if (lane == 0) red[wave][j] = v;
    }
    __syncthreads();
    if ((int)threadIdx.x < kRowRoutes && j0 + (int)threadIdx.x < a.top_k) {
        float v = red[0][threadIdx.x];
        for (int w = 1; w < waves; ++w) v += red[w][threadIdx.x];
        a.dweights[t * a.top_k + j0 + threadIdx.x] = v;
    }
    __syncthreads();
}

template <int TOKEN, int ROW>
__device__ __forceinline__ void scatter_rows(const MoeRowsArgs& a) {
    __shared__ float red[16][kRowRoutes];
    const int64_t t = a.token0 + blockIdx.x;
    const int H = a.hidden;
    for (int j0 = 0; j0 < a.top_k; j0 += kRowRoutes) {
        int slot[kRowRoutes];
        float w[kRowRoutes], d[kRowRoutes];
        row_routes(a, t, j0, slot, w);
#pragma unroll
        for (int j = 0; j < kRowRoutes; ++j) d[j] = 0.0f;
        for (int c = 8 * threadIdx.x; c < H; c += 8 * blockDim.x) {
            const int n = H - c;
            float v[8], y[kRowRoutes][8];
            row_load8<TOKEN>(a.tokens, t * H + c, n, v);
            if (a.dweights) {
#pragma unroll
                for (int j = 0; j < kRowRoutes; ++j)
                    if (slot[j] >= 0) row_load8<ROW>(a.rows_in, (int64_t)slot[j] * H + c, n, y[j]);
#pragma unroll
                for (int j = 0; j < kRowRoutes; ++j)
                    if (slot[j] >= 0) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) d[j] = __builtin_fmaf(y[j][i], v[i], d[j]);
                    }
            }
#pragma unroll
            for (int j = 0; j < kRowRoutes; ++j)
                if (slot[j] >= 0) {
                    float o[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[i] = a.weights ? w[j] * v[i] : v[i];
                    row_store8<ROW>(a.rows_out, (int64_t)slot[j] * H + c, n, o);
                }
        }
        if (a.dweights) row_dweights(a, t, j0, d, red);
    }
}

template <int TOKEN, int ROW>
__device__ __forceinline__ void gather_rows(const MoeRowsArgs& a) {
    __shared__ float red[16][kRowRoutes];
    const int64_t t = a.token0 + blockIdx.x;
    const int H = a.hidden;
    if (a.dweights) {
        for (int j0 = 0; j0 < a.top_k; j0 += kRowRoutes) {
            int slot[kRowRoutes];
            float w[kRowRoutes], d[kRowRoutes];
            row_routes(a, t, j0, slot, w);
#pragma unroll
            for (int j = 0; j < kRowRoutes; ++j) d[j] = 0.0f;
            for (int c = 8 * threadIdx.x; c < H; c += 8 * blockDim.x) {
                float v[8];
                row_load8<TOKEN>(a.dot, t * H + c, H - c, v);
#pragma unroll
                for (int j = 0; j < kRowRoutes; ++j)
                    if (slot[j] >= 0) {
                        float y[8];
                        row_load8<ROW>(a.rows_in, (int64_t)slot[j] * H + c, H - c, y);
#pragma unroll
                        for (int i = 0; i < 8; ++i) d[j] = __builtin_fmaf(y[i], v[i], d[j]);
                    }
            }
            row_dweights(a, t, j0, d, red);
        }
    }
    for (int c = 8 * threadIdx.x; c < H; c += 8 * blockDim.x) {
        const int n = H - c;
        float sum[8];
        if (a.shared) {
            row_load8<TOKEN>(a.shared, t * H + c, n, sum);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] = 0.0f;
        }
        for (int j0 = 0; j0 < a.top_k; j0 += kRowRoutes) {
            int slot[kRowRoutes];
            float w[kRowRoutes], y[kRowRoutes][8];
            row_routes(a, t, j0, slot, w);
#pragma unroll
            for (int j = 0; j < kRowRoutes; ++j)
                if (slot[j] >= 0) row_load8<ROW>(a.rows_in, (int64_t)slot[j] * H + c, n, y[j]);
#pragma unroll
            for (int j = 0; j < kRowRoutes; ++j)
                if (slot[j] >= 0) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) sum[i] = a.weights ? __builtin_fmaf(w[j], y[j][i], sum[i]) : sum[i] + y[j][i];
                }
        }
        row_store8<TOKEN>(a.out, t * H + c, n, sum);
    }
}

}  // namespace

#define NH_ROWS_KERNELS(name, body)                                                                                     \
    extern "C" __global__ __launch_bounds__(512) void nh_moe_##name##_f32_f32_kernel(MoeRowsArgs a) { body<DT_F32, DT_F32>(a); } \
    extern "C" __global__ __launch_bounds__(512) void nh_moe_##name##_f32_bf16_kernel(MoeRowsArgs a) { body<DT_F32, DT_BF16>(a); } \
    extern "C" __global__ __launch_bounds__(512) void nh_moe_##name##_bf16_f32_kernel(MoeRowsArgs a) { body<DT_BF16, DT_F32>(a); } \
    extern "C" __global__ __launch_bounds__(512) void nh_moe_##name##_bf16_bf16_kernel(MoeRowsArgs a) { body<DT_BF16, DT_BF16>(a); }
NH_ROWS_KERNELS(scatter_rows, scatter_rows)  // tokens' type, rows' type
NH_ROWS_KERNELS(gather_rows, gather_rows)
#undef NH_ROWS_KERNELS
