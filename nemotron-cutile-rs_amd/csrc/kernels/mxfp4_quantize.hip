// MXFP4 conversion kernels: rows to codes and back, weights and activations
// into the operand order of the products.
//
// A block's scale depends on its own 32 values only, so nothing here reduces
// over a row: four lanes share a block, eight values each (one 16-byte load of
// bf16, two of f32), and meet in two lane moves.  HBM-bound streaming work.
// The conversions are v_cvt_scalef32_pk_fp4_{f32,bf16} (round to nearest even,
// saturating, the scale's exponent subtracted): bit-identical to mx_code for
// every bf16 value under every scale byte a block of it can have, and on 2^24
// f32 values of all exponents with ties, checked on the device.
// 16384 x 4096 f32: to codes 57 us and back 54 (304 MB each: 5.3 and 5.6 TB/s),
// their codes into the tiled form 14 (71 MB, 5.1 TB/s); 613 x 2701 bf16, rows that
// start off alignment, 4.7 and 4.5; a row of 4096 2.5 and 2.3, which is a launch.
#include "mxfp4_device.h"

using namespace nh;

// One unit (eight values) per thread and turn, kTurns units in flight.
constexpr int kMxTurns = 4;

extern "C" __global__ __launch_bounds__(256) void nh_quantize_mxfp4_kernel(MxQuantizeArgs a) {
    const int64_t u0 = (int64_t)blockIdx.x * (256 * kMxTurns) + threadIdx.x;
    v4i v[kMxTurns][2];
    int count[kMxTurns];
    int64_t value[kMxTurns], code[kMxTurns], block[kMxTurns];
#pragma unroll
    for (int t = 0; t < kMxTurns; ++t) {
        const int64_t u = u0 + t * 256;
        count[t] = 0;
        value[t] = code[t] = block[t] = 0;
        if (u < a.units) {
            if (a.flat) {
                count[t] = 8;
                value[t] = u * 8;
                code[t] = u * 4;
                block[t] = u >> 2;
            } else {
                const int64_t row = a.units < (int64_t)1 << 32 ? (int64_t)((uint32_t)u / a.row_units) : u / a.row_units;
                const uint32_t c = (uint32_t)(u - row * a.row_units) * 8;
                count[t] = c < a.cols ? (int)min(8u, a.cols - c) : 0;
                value[t] = row * a.cols + c;
                code[t] = row * (int64_t)((a.cols + 1) / 2) + c / 2;
                block[t] = row * (a.row_units >> 2) + (c >> 5);
            }
        }
        mx_load8<true>(a.x, value[t], count[t], a.x_dtype, v[t]);
    }
#pragma unroll
    for (int t = 0; t < kMxTurns; ++t) {
        const int64_t u = u0 + t * 256;
        const uint32_t e = mx_scale_byte(quad_max_u32(mx_amax8(v[t], a.x_dtype)));
        if (e == kMxNan && a.nonfinite) mx_report8(a.nonfinite, kStageInput, value[t], count[t], a.x_dtype, v[t]);
        const uint32_t q = mx_encode8(v[t], e, a.x_dtype);
        if (count[t] == 8)
            __builtin_memcpy(a.codes + code[t], &q, 4);
        else
            for (int i = 0; i < (count[t] + 1) / 2; ++i) a.codes[code[t] + i] = (uint8_t)(q >> (8 * i));
        if (u < a.units && (threadIdx.x & 3) == 0) a.scales[block[t]] = (uint8_t)e;
    }
}

// 16 rows x 512 columns (one scale piece) per workgroup.  ONCE (many rows): past
// the caches, which then keep the codes for the product (2048 x 4096 -> 21504:
// 111.0 us, 112.9 without; 512 x 4096 -> 4096, where x itself is still there: 14.0
// against 13.6).  Rows are read whole
// waves at a time (1 KiB of bf16), the codes meet in LDS in tile order and
// leave as whole tiles (or 256 bytes of a row in the token form).
// (256 of the workgroup's threads, `tid` of them; every thread of the workgroup
// calls it, for one barrier.)
template <bool ONCE>
__device__ __forceinline__ void mx_quantize_tiles(const MxQuantizeTilesArgs& a, int64_t block, int tid, uint32_t* codes,
                                                  uint8_t* scales) {
    const int lane = tid & 63, wave = tid >> 6;
    const int64_t rt = block / a.kq;
    const int q = (int)(block - rt * a.kq);
    const int c = q * 512 + lane * 8;
    v4i v[4][2];
    int count[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = rt * 16 + wave * 4 + i;
        count[i] = row < a.rows && c < a.cols ? min(8, a.cols - c) : 0;
        mx_load8<ONCE>(a.x, row * a.cols + c, count[i], a.x_dtype, v[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = wave * 4 + i, b = lane >> 2;  // block b of the piece: K tile b / 4, lane group b % 4
        const uint32_t e = mx_scale_byte(quad_max_u32(mx_amax8(v[i], a.x_dtype)));
        if (e == kMxNan && a.nonfinite)
            mx_report8(a.nonfinite, kStageInput, (rt * 16 + r) * a.cols + c, count[i], a.x_dtype, v[i]);
        codes[(b * 16 + r) * 4 + (lane & 3)] = mx_encode8(v[i], e, a.x_dtype);
        if ((lane & 3) == 0) scales[((b & 3) * 16 + r) * 4 + (b >> 2)] = (uint8_t)e;
    }
    __syncthreads();
    const int live = min(4, a.kt - 4 * q);  // K tiles of this piece
    if (!a.token) {
        uint8_t* region = a.out + rt * ((int64_t)a.kt * 1024 + a.kq * 256);
        if (wave < live) *(v4i*)(region + (int64_t)(4 * q + wave) * 1024 + lane * 16) = *(const v4i*)(codes + tid * 4);
        if (tid < 64) *(uint32_t*)(region + (int64_t)a.kt * 1024 + q * 256 + tid * 4) = *(const uint32_t*)(scales + tid * 4);
    } else {
        const int r = tid >> 4, b = tid & 15;
        const int64_t row = rt * 16 + r;
        if (row < a.rows && (b >> 2) < live)
            *(v4i*)(a.out + row * ((int64_t)a.kt * 64) + q * 256 + b * 16) = *(const v4i*)(codes + (b * 16 + r) * 4);
        const int rs = tid >> 2, g = tid & 3;
        if (tid < 64 && rt * 16 + rs < a.rows)
            *(uint32_t*)(a.scales + (rt * 16 + rs) * ((int64_t)a.kq * 16) + q * 16 + g * 4) =
                *(const uint32_t*)(scales + (g * 16 + rs) * 4);
    }
}

extern "C" __global__ __launch_bounds__(256) void nh_quantize_mxfp4_tiles_kernel(MxQuantizeTilesArgs a) {
    __shared__ __align__(16) uint32_t codes[4 * 256];  // [K tile][lane][4]
    __shared__ __align__(4) uint8_t scales[256];       // [lane][K tile]
    if (a.once)
        mx_quantize_tiles<true>(a, blockIdx.x, threadIdx.x, codes, scales);
    else
        mx_quantize_tiles<false>(a, blockIdx.x, threadIdx.x, codes, scales);
}

// Codes and scales back to values: exact in f32, and in bf16 (two significant
// bits) wherever 6 * 2^127 does not overflow; a scale byte of 255 is NaN.
extern "C" __global__ __launch_bounds__(256) void nh_dequantize_mxfp4_kernel(MxDequantizeArgs a) {
    const int64_t u0 = (int64_t)blockIdx.x * (256 * kMxTurns) + threadIdx.x;
    uint32_t q[kMxTurns], e[kMxTurns];
    int count[kMxTurns];
    int64_t value[kMxTurns];
#pragma unroll
    for (int t = 0; t < kMxTurns; ++t) {
        const int64_t u = u0 + t * 256;
        int64_t code = 0, block = 0;
        count[t] = 0;
        value[t] = 0;
        q[t] = e[t] = 0;
        if (u >= a.units) continue;
        if (a.flat) {
            count[t] = 8;
            value[t] = u * 8;
            code = u * 4;
            block = u >> 2;
        } else {
            const int64_t row = a.units < (int64_t)1 << 32 ? (int64_t)((uint32_t)u / a.row_units) : u / a.row_units;
            const uint32_t c = (uint32_t)(u - row * a.row_units) * 8;
            count[t] = c < a.cols ? (int)min(8u, a.cols - c) : 0;
            value[t] = row * a.cols + c;
            code = row * (int64_t)((a.cols + 1) / 2) + c / 2;
            block = row * (a.row_units >> 2) + (c >> 5);
        }
        if (count[t] == 8)
            __builtin_memcpy(&q[t], a.codes + code, 4);
        else
            for (int i = 0; i < (count[t] + 1) / 2; ++i) q[t] |= (uint32_t)a.codes[code + i] << (8 * i);
        if (count[t]) e[t] = a.scales[block];
    }
#pragma unroll
    for (int t = 0; t < kMxTurns; ++t) {
        float v[8];
        mx_decode8(q[t], e[t], v);
        if (count[t] == 8) {
            if (a.out_dtype == DT_BF16) {
                const v4i w = {(int)f32x2_to_bf16x2(v[0], v[1]), (int)f32x2_to_bf16x2(v[2], v[3]),
                               (int)f32x2_to_bf16x2(v[4], v[5]), (int)f32x2_to_bf16x2(v[6], v[7])};
                __builtin_memcpy((uint16_t*)a.out + value[t], &w, 16);
            } else {
                __builtin_memcpy((float*)a.out + value[t], v, 32);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < count[t]) store_out(a.out, value[t] + i, v[i], a.out_dtype);
        }
    }
}

// Row-major codes and scales -> tiled form, one lane of four K tiles (64 bytes
// of codes, four scale bytes) per thread.
extern "C" __global__ __launch_bounds__(256) void nh_tile_mxfp4_kernel(MxTileArgs a) {
    const int64_t step = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.lanes; i += step) {
        const int lane = (int)(i & 63), g = lane >> 4;
        const int64_t piece = i >> 6, rt = piece / a.kq;
        const int q = (int)(piece - rt * a.kq);
        const int64_t row = rt * 16 + (lane & 15);
        uint8_t* region = a.tiled + rt * ((int64_t)a.kt * 1024 + a.kq * 256);
        const uint8_t* rc = a.codes + row * ((a.k + 1) / 2);
        const uint8_t* rs = a.scales + row * ((a.k + 31) / 32);
        uint32_t s = 0;
        for (int j = 0; j < 4 && 4 * q + j < a.kt; ++j) {
            const int c = (4 * q + j) * 128 + g * 32;
            v4i w = {0, 0, 0, 0};
            const int count = row < a.n && c < a.k ? min(32, a.k - c) : 0;
            if (count == 32) {
                __builtin_memcpy(&w, rc + c / 2, 16);
            } else {
                uint32_t t[4] = {0, 0, 0, 0};
                for (int b = 0; b < count; ++b) {  // the matrix edge, nibble by nibble: nothing past k
                    const uint32_t nib = (rc[(c + b) / 2] >> (4 * (b & 1))) & 15u;
#pragma unroll
                    for (int d = 0; d < 4; ++d)
                        if (d == b >> 3) t[d] |= nib << (4 * (b & 7));
                }
                w = v4i{(int)t[0], (int)t[1], (int)t[2], (int)t[3]};
            }
            if (count) s |= (uint32_t)rs[c / 32] << (8 * j);
            *(v4i*)(region + (int64_t)(4 * q + j) * 1024 + lane * 16) = w;
        }
        *(uint32_t*)(region + (int64_t)a.kt * 1024 + q * 256 + lane * 4) = s;
    }
}

// The MoE layer ahead of its experts, in one launch: workgroups of 16 waves
// route a token per wave (nh_moe_route_sigmoid_topk), the others quantize the
// tokens into the token form; neither waits for the other.  With few routes the
// one that routes also sorts them by expert (nh_moe_permute: stable, by route
// id), every thread counting against all routes in LDS.
extern "C" __global__ __launch_bounds__(1024) void nh_mx_moe_prep_kernel(MxMoePrepArgs a) {
    __shared__ __align__(16) uint32_t codes[4][4 * 256];
    __shared__ __align__(4) uint8_t scales[4][256];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if ((int)blockIdx.x >= a.route_blocks) {  // uniform
        const int64_t block = ((int64_t)blockIdx.x - a.route_blocks) * 4 + (tid >> 8);
        mx_quantize_tiles<false>(a.q, block, tid & 255, codes[tid >> 8], scales[tid >> 8]);  // past the rows: nothing
        return;
    }
    for (int token = (int)blockIdx.x * 16 + wave; token < a.r.tokens; token += 16 * a.route_blocks) {
        if (a.r.experts <= 128)
            route_kernel_body<2>(a.r, token, lane);
        else if (a.r.experts <= 256)
            route_kernel_body<4>(a.r, token, lane);
        else
            route_kernel_body<kMaxExpertsPerLane>(a.r, token, lane);
    }
    if (!a.permute) return;
    __syncthreads();  // the routes' stores are done
    const int R = a.p.routes, E = a.p.experts;
    int* ids = (int*)codes;
    if (tid < R) ids[tid] = a.p.indices[tid];
    __syncthreads();
    if (tid < R) {  // routing gives ids in [0, E)
        const int e = ids[tid];
        int slot = 0;
        for (int i = 0; i < R; ++i) slot += ids[i] < e || (ids[i] == e && i < tid);
        a.p.pos[tid] = slot;
        a.p.perm[slot] = tid;
    }
    for (int e = tid; e <= E; e += 1024) {
        int n = 0;
        for (int i = 0; i < R; ++i) n += ids[i] < e;
        a.p.offsets[e] = n;
    }
}
