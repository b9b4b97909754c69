// MXFP4 products of few rows, bound by the weight bytes: y = Q(x) W^T.
//
// A workgroup walks a run of 16-column weight tiles.  Its waves come in groups
// that take the run's tiles in turn, W waves to a group that split K: wave w
// owns the C K tiles [w C, w C + C) of every tile, keeps its part of the
// activations in registers as MFMA operands for the whole run, and has the
// weights of D column tiles in flight.  The waves' partial tiles meet in LDS
// (f32), one barrier per unit, two buffers.  The MX blocks make the activation
// side local: lane (g, r) of a K tile needs 32 consecutive values of row r,
// which are one block with one scale, so a wave quantizes exactly what it
// multiplies, in place, with no reduction, no exchange and no barrier.  The
// activations' loads go out ahead of the weights', so their quantization runs
// under the weights' latency.
//
// Forms: the activations as f32 / bf16 rows (up to 16, quantized here) or codes
// in the token form (up to 16 RB rows, gathered through a permutation); the
// output as f32 / bf16 rows with a bias, or ReLU^2 of it quantized again in
// units of two column tiles (one block of 32), in the token form that the next
// product gathers; one product, or one per expert over the routes' segments.
//
// One row of 4096 -> 16384 takes 9.8 us (36 MB), eight of 4096 -> 131072 47
// (289 MB, 6.1 TB/s); 128 experts of 2688 x 1856 reached by 500 tokens, 6 routes
// each, 70 us up and 73 down (342 MB each, 4.9 and 4.7 TB/s).  Rows of any
// alignment, of f32 past K = 4096 or of bf16 past 8192 issue the weights behind
// their quantization: 8 x 2701 -> 4099 10.5 us, 1 x 8192 f32 -> 4096 16, 1 x 16384
// -> 4096 30.
#include "mxfp4_device.h"

using namespace nh;

namespace {

enum { kMxTokens, kMxRowsBf16, kMxRowsF32, kMxRowsAny };  // activations
enum { kMxOut, kMxRequant };                              // output

// A wave's place, and its workgroup's run of units.
struct MxPlace {
    int lane, wave, group, W, groups;
    int seg0, seg1;            // rows (slots) of the product
    int u_begin, u_end;
    const uint8_t* w;          // the product's weights
    const float* bias;         // and bias
    uint32_t region;
    int ntiles;
};

// The first non-finite value of this lane's blocks of row m, read again (rare),
// into the caller's word; by one workgroup, every one of them reads the rows.
template <int C>
__device__ __forceinline__ void mx_report_rows(const MxStreamArgs& a, const MxPlace& p, int m) {
    if (!a.nonfinite || blockIdx.x != 0 || p.group != 0) return;
#pragma unroll 1
    for (int i = 0; i < C * 32; ++i) {
        const int k = (p.wave * C + (i >> 5)) * 128 + (p.lane >> 4) * 32 + (i & 31);
        if (k >= a.K) break;
        const float f = load_as_f32(a.x, (int64_t)m * a.K + k, a.x_dtype);
        if (is_finite_f32(f)) continue;
        report_nonfinite(a.nonfinite, kStageInput, (int64_t)m * a.K + k, f);
        break;
    }
}

// The operands of a wave's C K tiles of 16 rows from row m0: the rows' blocks
// are loaded CC K tiles at a time, `start` issues the weights behind the first.
template <int C, int DT, class Start>
__device__ __forceinline__ void mx_rows_operand(const MxStreamArgs& a, const MxPlace& p, int m0, v4i (&x)[C],
                                                int (&xs)[(C + 3) / 4], Start start) {
    constexpr int NV = DT == DT_BF16 ? 4 : 8;          // 16-byte loads per block
    constexpr int CC = C * NV <= 16 ? C : 16 / NV;     // at most 16 of them
    constexpr int esz = DT == DT_BF16 ? 2 : 4;
    const int m = m0 + (p.lane & 15), g = p.lane >> 4;
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(a.x, (uint32_t)a.M * (uint32_t)a.K * esz);
    bool bad = false;
#pragma unroll
    for (int s = 0; s < (C + 3) / 4; ++s) xs[s] = 0;
#pragma unroll
    for (int c0 = 0; c0 < C; c0 += CC) {
        v4i v[CC][NV];
#pragma unroll
        for (int c = 0; c < CC; ++c) {
            const int k = (p.wave * C + c0 + c) * 128 + g * 32;
            const int off = m < a.M && k < a.K ? (m * a.K + k) * esz : kOutOfRange - 16 * NV;
#pragma unroll
            for (int j = 0; j < NV; ++j) v[c][j] = buffer_load16(rs, off + 16 * j);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (c0 == 0) start();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int c = 0; c < CC; ++c) {
            uint32_t amax = 0;
#pragma unroll
            for (int j = 0; j < NV; ++j) amax = DT == DT_BF16 ? absbits_bf16x8(v[c][j], amax) : absbits_f32x4(v[c][j], amax);
            const uint32_t e = mx_scale_byte(DT == DT_BF16 ? absbits_pair_f32(amax) : amax);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (DT == DT_BF16) {
                    x[c0 + c][j] = (int)mx_encode_bf16x8(v[c][j], e);
                } else {
                    float f[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) f[i] = f32_from_bits((uint32_t)v[c][2 * j + (i >> 2)][i & 3]);
                    x[c0 + c][j] = (int)mx_encode_f32x8(f, e);
                }
            }
            xs[(c0 + c) >> 2] |= (int)(e << (8 * ((c0 + c) & 3)));
            bad |= e == kMxNan;
        }
    }
    if (bad) mx_report_rows<C>(a, p, m);
}

// The same for rows of any alignment and width, value by value at the edge: a
// loop over the K tiles (unrolled, its branches are many times the rest).
template <int C>
__device__ __forceinline__ void mx_rows_operand_any(const MxStreamArgs& a, const MxPlace& p, int m0, v4i (&x)[C],
                                                    int (&xs)[(C + 3) / 4]) {
    const int m = m0 + (p.lane & 15), g = p.lane >> 4;
    bool bad = false;
#pragma unroll
    for (int s = 0; s < (C + 3) / 4; ++s) xs[s] = 0;
#pragma unroll
    for (int c = 0; c < C; ++c) x[c] = v4i{0, 0, 0, 0};
#pragma unroll 1
    for (int c = 0; c < C; ++c) {
        const int k = (p.wave * C + c) * 128 + g * 32;
        const int count = m < a.M && k < a.K ? min(32, a.K - k) : 0;
        v4i v[4][2];
        uint32_t amax = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            mx_load8(a.x, (int64_t)m * a.K + k + 8 * j, max(0, min(8, count - 8 * j)), a.x_dtype, v[j]);
            amax = max(amax, mx_amax8(v[j], a.x_dtype));
        }
        const uint32_t e = mx_scale_byte(amax);
        bad |= e == kMxNan;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int q = (int)mx_encode8(v[j], e, a.x_dtype);
#pragma unroll
            for (int t = 0; t < C; ++t)
                if (t == c) x[t][j] = q;
        }
#pragma unroll
        for (int s = 0; s < (C + 3) / 4; ++s)
            if (s == c >> 2) xs[s] |= (int)(e << (8 * (c & 3)));
    }
    if (bad) mx_report_rows<C>(a, p, m);
}

// The run of column tiles over rows m0 .. m0 + 16 RB - 1 (below p.seg1).
template <int C, int RB, int D, int SRC, int EPI>
__device__ __forceinline__ void mx_pass(const MxStreamArgs& a, const MxPlace& p, int m0, int8_t* lds) {
    constexpr int T = EPI == kMxRequant ? 2 : 1;  // column tiles per unit
    constexpr int CS = (C + 3) / 4;               // scale dwords per tile
    const int lane = p.lane, r16 = lane & 15, g = lane >> 4, W = p.W;
    const int kt0 = p.wave * C;
    const int rounds = (p.u_end - p.u_begin + p.groups - 1) / p.groups, steps = rounds * T;
    v4f* red = (v4f*)lds + (size_t)p.group * (2 * T * RB * W * 64);             // [2][T][RB][W][64]
    const float* sbias = (const float*)(lds + (size_t)2 * T * RB * W * p.groups * 1024);  // of the run
    // tile of step s: unit u_begin + group + (s / T) groups
    auto tile_of = [&](int s) { return (p.u_begin + p.group + (s / T) * p.groups) * T + (T == 2 ? s & 1 : 0); };

    // weights of step s, this wave's K tiles (zeros past the matrix)
    v4i w[D][C];
    int ws[D][CS];
    auto load = [&](int d, int s) {
        const int t = tile_of(s);
        const bool live = t < p.u_end * T && t < p.ntiles;
        const __amdgpu_buffer_rsrc_t rs = make_rsrc(p.w + (int64_t)t * p.region, live ? p.region : 0u);
#pragma unroll
        for (int c = 0; c < C; ++c)
            w[d][c] = buffer_load16_stream(rs, kt0 + c < a.kt ? (kt0 + c) * 1024 + lane * 16 : kOutOfRange);
#pragma unroll
        for (int s4 = 0; s4 < CS; ++s4)
            ws[d][s4] = __builtin_amdgcn_raw_buffer_load_b32(rs, a.kt * 1024 + ((kt0 >> 2) + s4) * 256 + lane * 4, 0, 0);
    };
    auto start = [&]() {
#pragma unroll
        for (int d = 0; d < D; ++d) load(d, d);
    };
    // activations: this wave's operands, byte c % 4 of scale dword c / 4
    v4i x[RB][C];
    int xs[RB][CS];
    // (kernels of their own: where branches meet, registers of loads in flight are moved, so waited for)
    static_assert(SRC == kMxTokens || RB == 1, "rows are quantized 16 at a time");
    if constexpr (SRC == kMxRowsAny) {
        mx_rows_operand_any<C>(a, p, m0, x[0], xs[0]);
        start();
    } else if constexpr (SRC == kMxRowsBf16) {
        mx_rows_operand<C, DT_BF16>(a, p, m0, x[0], xs[0], start);
    } else if constexpr (SRC == kMxRowsF32) {
        mx_rows_operand<C, DT_F32>(a, p, m0, x[0], xs[0], start);
    } else {
        int64_t row[RB];
        bool ok[RB];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const int slot = m0 + rb * 16 + r16;
            ok[rb] = slot < p.seg1;
            row[rb] = !ok[rb] ? 0 : a.perm ? a.perm[slot] / a.gather_div : slot;
        }
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const uint8_t* xc = a.xcodes + row[rb] * ((int64_t)a.kt * 64) + g * 16;
            const uint8_t* xsc = a.xscales + row[rb] * ((int64_t)a.kq * 16) + g * 4;
#pragma unroll
            for (int c = 0; c < C; ++c)
                x[rb][c] = ok[rb] && kt0 + c < a.kt ? *(const v4i*)(xc + (kt0 + c) * 64) : v4i{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < CS; ++s)
                xs[rb][s] = ok[rb] && (kt0 >> 2) + s < a.kq ? *(const int*)(xsc + ((kt0 >> 2) + s) * 16) : 0;
        }
        __builtin_amdgcn_sched_barrier(0);
        start();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int s = 0; s < CS; ++s) {
                // bytes of K tiles past the last are not written by a requantizing product
                const int bytes = a.kt - 4 * ((kt0 >> 2) + s);  // uniform
                if (bytes < 4) xs[rb][s] &= bytes > 0 ? (1 << (8 * bytes)) - 1 : 0;
                // a wave of two K tiles may start inside a dword
                if constexpr (C < 4) xs[rb][s] = (int)((uint32_t)xs[rb][s] >> (8 * (kt0 & 3)));
            }
    }
    int buf = 0;
    for (int sb = 0; sb < steps; sb += D) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            const int s = sb + d;
            // Uniform.  Not a break: where that joins the back edge the compiler
            // would count no earlier load as in flight, and wait for all of them.
            const bool live = s < steps;
            v4f acc[RB];
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) acc[rb] = v4f{0.f, 0.f, 0.f, 0.f};
            if constexpr (C < 4) ws[d][0] = (int)((uint32_t)ws[d][0] >> (8 * (kt0 & 3)));
            if (live) {
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
            }
            load(d, s + D);
            if (!live) continue;
            const int h = T == 1 ? 0 : s & 1;
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) red[((((buf * T + h) * RB) + rb) * W + p.wave) * 64 + lane] = acc[rb];
            if (T == 2 && h == 0) continue;  // the unit's other half
            lds_publish();
            const int u = p.u_begin + p.group + (s / T) * p.groups;
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                // (a group past the run's last unit has no outputs, and no bias in LDS)
                if (u >= p.u_end || ((s / T) * RB + rb) % W != p.wave) continue;
                const int row = m0 + rb * 16 + r16;
                float y[T][4];
#pragma unroll
                for (int i = 0; i < T; ++i) {
                    const v4f* part = red + ((((buf * T + i) * RB) + rb) * W) * 64 + lane;
                    v4f q[8];  // every read in flight
#pragma unroll
                    for (int v = 0; v < 8; ++v) q[v] = part[min(v, W - 1) * 64];
                    v4f sum = q[0];
#pragma unroll
                    for (int v = 1; v < 8; ++v)
                        if (v < W) sum += q[v];
                    const int ln = (u * T + i) * 16 + 4 * g - p.u_begin * T * 16;
#pragma unroll
                    for (int n = 0; n < 4; ++n) y[i][n] = a.bias ? sum[n] + sbias[ln + n] : sum[n];
                }
                if (row >= p.seg1) continue;
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
                    const uint32_t e = mx_scale_byte(amax);
                    if (e == kMxNan && a.nonfinite)
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (!is_finite_f32(v[i]))
                                report_nonfinite(a.nonfinite, a.nonfinite_stage,
                                                 (int64_t)row * a.N + n + 16 * (i >> 2) + (i & 3), v[i]);
                    const uint32_t q = mx_encode_f32x8(v, e);
                    const int hkt = (a.N + 127) >> 7, hkq = (hkt + 3) >> 2, kt = u >> 2, hg = u & 3;
                    uint8_t* hc = a.hcodes + row * ((int64_t)hkt * 64) + u * 16;
                    *(uint16_t*)(hc + 2 * g) = (uint16_t)q;
                    *(uint16_t*)(hc + 8 + 2 * g) = (uint16_t)(q >> 16);
                    if (g == 0) a.hscales[row * ((int64_t)hkq * 16) + (kt >> 2) * 16 + hg * 4 + (kt & 3)] = (uint8_t)e;
                }
            }
            buf ^= 1;
        }
    }
}

template <int C, int RB, int D, int SRC, int EPI>
__device__ __forceinline__ void mx_stream(const MxStreamArgs& a, int8_t* lds) {
    constexpr int T = EPI == kMxRequant ? 2 : 1;
    MxPlace p;
    p.lane = threadIdx.x & 63;
    p.W = a.waves;
    p.groups = a.groups;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    p.group = wave / p.W;
    p.wave = wave - p.group * p.W;
    int e = 0;
    p.seg0 = 0;
    p.seg1 = a.M;
    if (a.offsets) {
        e = (int)(blockIdx.y / (unsigned)a.row_parts);
        if (a.compact) {
            e = nth_active_expert(a.offsets, a.experts, e, p.lane, p.seg0, p.seg1);
        } else {
            p.seg0 = a.offsets[e];
            p.seg1 = a.offsets[e + 1];
            if (p.seg0 >= p.seg1) e = -1;
        }
        if (e < 0) return;  // uniform: no routes
    }
    // the run: the first `longer` workgroups take one unit more
    const int b = blockIdx.x;
    p.u_begin = b * a.run + min(b, a.longer);
    p.u_end = p.u_begin + a.run + (b < a.longer ? 1 : 0);
    p.ntiles = (a.N + 15) >> 4;
    p.region = (uint32_t)a.kt * 1024u + (uint32_t)a.kq * 256u;
    p.w = a.w + (int64_t)e * p.ntiles * p.region;
    if (a.bias) {  // of the run, behind the partial tiles
        float* sbias = (float*)(lds + (size_t)2 * T * a.row_blocks * p.W * p.groups * 1024);
        for (int i = threadIdx.x; i < (p.u_end - p.u_begin) * T * 16; i += blockDim.x) {
            const int n = p.u_begin * T * 16 + i;
            sbias[i] = n < a.N ? a.bias[(int64_t)e * a.N + n] : 0.0f;
        }
    }
    // workgroups of an expert's row parts take its passes in turn
    const int step = 16 * RB * a.row_parts;
    for (int m0 = p.seg0 + 16 * RB * (int)(blockIdx.y % (unsigned)a.row_parts); m0 < p.seg1; m0 += step) {
        mx_pass<C, RB, D, SRC, EPI>(a, p, m0, lds);
        if (m0 + step < p.seg1) lds_publish();  // the last sums are read before the next pass writes partials
    }
}

}  // namespace

#define NH_MX_STREAM(name, C, RB, D, SRC, EPI)                                        \
    extern "C" __global__ __launch_bounds__(512, 2) void name(MxStreamArgs a) {       \
        extern __shared__ __align__(1024) int8_t lds[];                               \
        mx_stream<C, RB, D, SRC, EPI>(a, lds);                                        \
    }
// rows quantized here (up to 16): K up to 1024, 4096, 8192, 16384; the straight
// forms whose loads fit the registers next to the weights in flight
NH_MX_STREAM(nh_mx_stream_bf16_2_kernel, 2, 1, 8, kMxRowsBf16, kMxOut)
NH_MX_STREAM(nh_mx_stream_bf16_4_kernel, 4, 1, 4, kMxRowsBf16, kMxOut)
NH_MX_STREAM(nh_mx_stream_bf16_8_kernel, 8, 1, 2, kMxRowsBf16, kMxOut)
NH_MX_STREAM(nh_mx_stream_f32_2_kernel, 2, 1, 8, kMxRowsF32, kMxOut)
NH_MX_STREAM(nh_mx_stream_f32_4_kernel, 4, 1, 4, kMxRowsF32, kMxOut)
NH_MX_STREAM(nh_mx_stream_any_2_kernel, 2, 1, 8, kMxRowsAny, kMxOut)
NH_MX_STREAM(nh_mx_stream_any_4_kernel, 4, 1, 4, kMxRowsAny, kMxOut)
NH_MX_STREAM(nh_mx_stream_any_8_kernel, 8, 1, 2, kMxRowsAny, kMxOut)
NH_MX_STREAM(nh_mx_stream_any_16_kernel, 16, 1, 1, kMxRowsAny, kMxOut)
// codes: 16 rows at once, 32, or 64 (of K up to 4096)
NH_MX_STREAM(nh_mx_stream_tok2_kernel, 2, 1, 8, kMxTokens, kMxOut)
NH_MX_STREAM(nh_mx_stream_tok4_kernel, 4, 1, 4, kMxTokens, kMxOut)
NH_MX_STREAM(nh_mx_stream_tok8_kernel, 8, 1, 2, kMxTokens, kMxOut)
NH_MX_STREAM(nh_mx_stream_tok2_32_kernel, 2, 2, 8, kMxTokens, kMxOut)
NH_MX_STREAM(nh_mx_stream_tok4_32_kernel, 4, 2, 4, kMxTokens, kMxOut)
NH_MX_STREAM(nh_mx_stream_tok8_32_kernel, 8, 2, 2, kMxTokens, kMxOut)
NH_MX_STREAM(nh_mx_stream_tok2_64_kernel, 2, 4, 8, kMxTokens, kMxOut)
NH_MX_STREAM(nh_mx_stream_tok4_64_kernel, 4, 4, 4, kMxTokens, kMxOut)
NH_MX_STREAM(nh_mx_stream_requant2_kernel, 2, 1, 8, kMxTokens, kMxRequant)
NH_MX_STREAM(nh_mx_stream_requant4_kernel, 4, 1, 4, kMxTokens, kMxRequant)
NH_MX_STREAM(nh_mx_stream_requant8_kernel, 8, 1, 2, kMxTokens, kMxRequant)
NH_MX_STREAM(nh_mx_stream_requant2_32_kernel, 2, 2, 8, kMxTokens, kMxRequant)
NH_MX_STREAM(nh_mx_stream_requant4_32_kernel, 4, 2, 4, kMxTokens, kMxRequant)
NH_MX_STREAM(nh_mx_stream_requant8_32_kernel, 8, 2, 2, kMxTokens, kMxRequant)
NH_MX_STREAM(nh_mx_stream_requant2_64_kernel, 2, 4, 4, kMxTokens, kMxRequant)
NH_MX_STREAM(nh_mx_stream_requant4_64_kernel, 4, 4, 2, kMxTokens, kMxRequant)
