// MXFP4 products of few rows, bound by the weight bytes: y = Q(x) W^T.
//
// A workgroup walks a run of 16-column weight tiles with W waves that split K:
// wave w owns the C K tiles [w C, w C + C) of every tile, keeps its part of the
// activations in registers as MFMA operands for the whole run, and has the
// weights of D column tiles in flight.  The waves' partial tiles of a unit meet
// in LDS (f32), one barrier per unit, two buffers.  The MX blocks make the
// activation side local: lane (g, r) of a K tile needs 32 consecutive values of
// row r, which are one block with one scale, so a wave quantizes exactly what
// it multiplies, in place, with no reduction, no exchange and no barrier.
//
// Forms: the activations as f32 / bf16 rows (up to 16, quantized here) or codes
// in the token form (up to 16 RB rows, gathered through a permutation); the
// output as f32 / bf16 rows with a bias, or ReLU^2 of it quantized again in
// units of two column tiles (one block of 32), in the token form that the next
// product gathers; one product, or one per expert over the routes' segments.
#include <type_traits>

#include "mxfp4_device.h"

using namespace nh;

namespace {

enum { kMxRows = 0, kMxTokens = 1 };            // activations
enum { kMxOut = 0, kMxRequant = 1 };            // output

// The expert of this workgroup's y, and its slots.
__device__ __forceinline__ int mx_expert(const MxStreamArgs& a, int lane, int& seg0, int& seg1) {
    int e = blockIdx.y;
    if (a.compact) return nth_active_expert(a.offsets, a.experts, e, lane, seg0, seg1);
    seg0 = a.offsets[e];
    seg1 = a.offsets[e + 1];
    return seg0 < seg1 ? e : -1;
}

template <int C, int RB, int D, int SRC, int EPI>
__device__ __forceinline__ void mx_stream(const MxStreamArgs& a, int8_t* lds) {
    constexpr int T = EPI == kMxRequant ? 2 : 1;  // column tiles per unit
    constexpr int CS = (C + 3) / 4;               // scale dwords per tile
    const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), W = blockDim.x >> 6;
    int e = 0, seg0 = 0, seg1 = a.M;
    if (a.offsets) {
        e = mx_expert(a, lane, seg0, seg1);
        if (e < 0) return;  // uniform: no routes
    }
    const int u_begin = (int)((int64_t)a.units * blockIdx.x / gridDim.x);
    const int u_end = (int)((int64_t)a.units * (blockIdx.x + 1) / gridDim.x);
    if (u_begin >= u_end) return;
    const int ntiles = (a.N + 15) >> 4;
    const uint32_t region = (uint32_t)a.kt * 1024u + (uint32_t)a.kq * 256u;
    const uint8_t* wexp = a.w + (int64_t)e * ntiles * region;
    const int kt0 = wave * C;
    v4f* red = (v4f*)lds;                                   // [2][T][RB][W][64]
    float* sbias = (float*)(lds + 2 * T * RB * W * 1024);   // [16 T (units of the run)]
    if (a.bias)
        for (int i = threadIdx.x; i < (u_end - u_begin) * T * 16; i += blockDim.x) {
            const int n = u_begin * T * 16 + i;
            sbias[i] = n < a.N ? a.bias[(int64_t)e * a.N + n] : 0.0f;
        }

    // weights of tile t, this wave's K tiles (zeros past the matrix)
    v4i w[D][C];
    int ws[D][CS];
    auto load = [&](int d, int t) {
        const bool live = t < u_end * T && t < ntiles;
        const __amdgpu_buffer_rsrc_t rs = make_rsrc(wexp + (int64_t)t * region, live ? region : 0u);
#pragma unroll
        for (int c = 0; c < C; ++c)
            w[d][c] = buffer_load16_stream(rs, kt0 + c < a.kt ? (kt0 + c) * 1024 + lane * 16 : kOutOfRange);
#pragma unroll
        for (int s = 0; s < CS; ++s)
            ws[d][s] = __builtin_amdgcn_raw_buffer_load_b32(rs, a.kt * 1024 + ((kt0 >> 2) + s) * 256 + lane * 4, 0, 0);
    };
    for (int p0 = seg0; p0 < seg1; p0 += 16 * RB) {
        // activations: this wave's operands, byte c % 4 of scale dword c / 4
        v4i x[RB][C];
        int xs[RB][CS];
        if constexpr (SRC == kMxRows) {
            static_assert(RB == 1, "rows are quantized 16 at a time");
            const int m = p0 + r16;
#pragma unroll
            for (int s = 0; s < CS; ++s) xs[0][s] = 0;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int k = (kt0 + c) * 128 + g * 32;
                const int count = m < seg1 && k < a.K ? min(32, a.K - k) : 0;
                v4i v[4][2];
                uint32_t amax = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    mx_load8(a.x, (int64_t)m * a.K + k + 8 * j, max(0, min(8, count - 8 * j)), a.x_dtype, v[j]);
                    amax = max(amax, mx_amax8(v[j], a.x_dtype));
                }
                const uint32_t eb = mx_scale_byte(amax);
                if (eb == kMxNan && a.nonfinite && blockIdx.x == 0)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        mx_report8(a.nonfinite, kStageInput, (int64_t)m * a.K + k + 8 * j, max(0, min(8, count - 8 * j)),
                                   a.x_dtype, v[j]);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[0][c][j] = (int)mx_encode8(v[j], eb, a.x_dtype);
                xs[0][c >> 2] |= (int)(eb << (8 * (c & 3)));
            }
        } else {
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                const int slot = p0 + rb * 16 + r16;
                const bool ok = slot < seg1;
                const int64_t row = !ok ? 0 : a.perm ? a.perm[slot] / a.gather_div : slot;
                const uint8_t* xc = a.xcodes + row * ((int64_t)a.kt * 64) + g * 16;
                const uint8_t* xsc = a.xscales + row * ((int64_t)a.kq * 16) + g * 4;
#pragma unroll
                for (int c = 0; c < C; ++c)
                    x[rb][c] = ok && kt0 + c < a.kt ? *(const v4i*)(xc + (kt0 + c) * 64) : v4i{0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < CS; ++s) {
                    // bytes of K tiles past the last are not written by a requantizing product
                    const int bytes = a.kt - 4 * ((kt0 >> 2) + s);  // uniform
                    xs[rb][s] = ok && bytes > 0 ? *(const int*)(xsc + ((kt0 >> 2) + s) * 16) : 0;
                    if (bytes < 4) xs[rb][s] &= bytes > 0 ? (1 << (8 * bytes)) - 1 : 0;
                }
            }
        }
        // a wave of fewer than four K tiles starts inside a scale dword
        if constexpr (C < 4 && SRC == kMxTokens) {
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) xs[rb][0] = (int)((uint32_t)xs[rb][0] >> (8 * (kt0 & 3)));
        }
        const int t0 = u_begin * T, t1 = u_end * T;
#pragma unroll
        for (int d = 0; d < D; ++d) load(d, t0 + d);
        int buf = 0;
        for (int tb = t0; tb < t1; tb += D) {
#pragma unroll
            for (int d = 0; d < D; ++d) {
                const int t = tb + d;
                if (t >= t1) break;  // uniform
                v4f acc[RB];
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) acc[rb] = v4f{0.f, 0.f, 0.f, 0.f};
                if constexpr (C < 4) ws[d][0] = (int)((uint32_t)ws[d][0] >> (8 * (kt0 & 3)));
#pragma unroll
                for (int c = 0; c < C; ++c)
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) {
                        const int sw = ws[d][c >> 2], sa = xs[rb][c >> 2];
                        if ((c & 3) == 0) acc[rb] = mx_mfma<0, 0>(w[d][c], x[rb][c], acc[rb], sw, sa);
                        if ((c & 3) == 1) acc[rb] = mx_mfma<1, 1>(w[d][c], x[rb][c], acc[rb], sw, sa);
                        if ((c & 3) == 2) acc[rb] = mx_mfma<2, 2>(w[d][c], x[rb][c], acc[rb], sw, sa);
                        if ((c & 3) == 3) acc[rb] = mx_mfma<3, 3>(w[d][c], x[rb][c], acc[rb], sw, sa);
                    }
                load(d, t + D);
                const int h = T == 1 ? 0 : t & 1;
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) red[((((buf * T + h) * RB) + rb) * W + wave) * 64 + lane] = acc[rb];
                if (T == 2 && h == 0) continue;  // the unit's other half (t0 is even)
                lds_publish();
                const int u = T == 1 ? t : t >> 1;
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    if ((u * RB + rb) % W != wave) continue;
                    const int row = p0 + rb * 16 + r16;
                    float y[T][4];
#pragma unroll
                    for (int i = 0; i < T; ++i) {
                        v4f sum = red[((((buf * T + i) * RB) + rb) * W) * 64 + lane];
                        for (int v = 1; v < W; ++v) sum += red[((((buf * T + i) * RB) + rb) * W + v) * 64 + lane];
                        const int ln = (u * T + i) * 16 + 4 * g - u_begin * T * 16;
#pragma unroll
                        for (int q = 0; q < 4; ++q) y[i][q] = a.bias ? sum[q] + sbias[ln + q] : sum[q];
                    }
                    if (row >= seg1) continue;
                    if constexpr (EPI == kMxOut) {
                        const int n = u * 16 + 4 * g;
                        const int64_t o = (int64_t)row * a.N + n;
                        if (n + 3 < a.N)
                            store_cols4((int8_t*)a.out + o * (a.out_dtype == DT_BF16 ? 2 : 4), y[0], a.out_dtype == DT_BF16);
                        else
#pragma unroll
                            for (int q = 0; q < 4; ++q)
                                if (n + q < a.N) store_out(a.out, o + q, y[0][q], a.out_dtype);
                    } else {
                        // ReLU^2, then the block of 32 columns that the four lanes of this row hold
                        const int n = u * 32 + 4 * g;
                        uint32_t amax = 0;
                        float v[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float t2 = y[i >> 2][i & 3];
                            // a NaN stays one here: it comes from a block with no value, and marks the next
                            v[i] = t2 != t2 ? t2 : relu2(t2);
                            if (n + 16 * (i >> 2) + (i & 3) >= a.N) v[i] = 0.0f;
                            amax = max(amax, f32_bits(v[i]) & 0x7fffffffu);
                        }
                        amax = max(amax, (uint32_t)__shfl_xor((int)amax, 16, kWave));
                        amax = max(amax, (uint32_t)__shfl_xor((int)amax, 32, kWave));
                        const uint32_t eb = mx_scale_byte(amax);
                        if (eb == kMxNan && a.nonfinite)
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                if (!is_finite_f32(v[i]))
                                    report_nonfinite(a.nonfinite, a.nonfinite_stage,
                                                     (int64_t)row * a.N + n + 16 * (i >> 2) + (i & 3), v[i]);
                        const uint32_t q = mx_encode_f32x8(v, eb);
                        const int hkt = (a.N + 127) >> 7, hkq = (hkt + 3) >> 2, kt = u >> 2, hg = u & 3;
                        uint8_t* hc = a.hcodes + row * ((int64_t)hkt * 64) + u * 16;
                        *(uint16_t*)(hc + 2 * g) = (uint16_t)q;
                        *(uint16_t*)(hc + 8 + 2 * g) = (uint16_t)(q >> 16);
                        if (g == 0) a.hscales[row * ((int64_t)hkq * 16) + (kt >> 2) * 16 + hg * 4 + (kt & 3)] = (uint8_t)eb;
                    }
                }
                buf ^= 1;
            }
        }
        if (p0 + 16 * RB < seg1) lds_publish();  // the last sums are read before the next pass writes partials
    }
}

}  // namespace

#define NH_MX_STREAM(name, C, RB, D, SRC, EPI)                                        \
    extern "C" __global__ __launch_bounds__(512, 2) void name(MxStreamArgs a) {       \
        extern __shared__ __align__(1024) int8_t lds[];                               \
        mx_stream<C, RB, D, SRC, EPI>(a, lds);                                        \
    }
// rows quantized here (up to 16): K up to 1024, 2048, 4096, 8192, 16384
NH_MX_STREAM(nh_mx_stream_rows1_kernel, 1, 1, 8, kMxRows, kMxOut)
NH_MX_STREAM(nh_mx_stream_rows2_kernel, 2, 1, 6, kMxRows, kMxOut)
NH_MX_STREAM(nh_mx_stream_rows4_kernel, 4, 1, 4, kMxRows, kMxOut)
NH_MX_STREAM(nh_mx_stream_rows8_kernel, 8, 1, 2, kMxRows, kMxOut)
NH_MX_STREAM(nh_mx_stream_rows16_kernel, 16, 1, 1, kMxRows, kMxOut)
// codes: up to 16 rows at once, or 64 (32 of K past 4096)
NH_MX_STREAM(nh_mx_stream_tok1_kernel, 1, 1, 8, kMxTokens, kMxOut)
NH_MX_STREAM(nh_mx_stream_tok2_kernel, 2, 1, 6, kMxTokens, kMxOut)
NH_MX_STREAM(nh_mx_stream_tok4_kernel, 4, 1, 4, kMxTokens, kMxOut)
NH_MX_STREAM(nh_mx_stream_tok8_kernel, 8, 1, 2, kMxTokens, kMxOut)
NH_MX_STREAM(nh_mx_stream_tok1_wide_kernel, 1, 4, 8, kMxTokens, kMxOut)
NH_MX_STREAM(nh_mx_stream_tok2_wide_kernel, 2, 4, 6, kMxTokens, kMxOut)
NH_MX_STREAM(nh_mx_stream_tok4_wide_kernel, 4, 4, 3, kMxTokens, kMxOut)
NH_MX_STREAM(nh_mx_stream_tok8_wide_kernel, 8, 2, 2, kMxTokens, kMxOut)
NH_MX_STREAM(nh_mx_stream_requant1_kernel, 1, 1, 8, kMxTokens, kMxRequant)
NH_MX_STREAM(nh_mx_stream_requant2_kernel, 2, 1, 6, kMxTokens, kMxRequant)
NH_MX_STREAM(nh_mx_stream_requant4_kernel, 4, 1, 4, kMxTokens, kMxRequant)
NH_MX_STREAM(nh_mx_stream_requant8_kernel, 8, 1, 2, kMxTokens, kMxRequant)
NH_MX_STREAM(nh_mx_stream_requant1_wide_kernel, 1, 4, 8, kMxTokens, kMxRequant)
NH_MX_STREAM(nh_mx_stream_requant2_wide_kernel, 2, 4, 6, kMxTokens, kMxRequant)
NH_MX_STREAM(nh_mx_stream_requant4_wide_kernel, 4, 4, 2, kMxTokens, kMxRequant)
NH_MX_STREAM(nh_mx_stream_requant8_wide_kernel, 8, 2, 2, kMxTokens, kMxRequant)
