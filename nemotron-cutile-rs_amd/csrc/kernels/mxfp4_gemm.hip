// MXFP4 product of many rows: both operands in the tiled form, streamed into an
// LDS ring and multiplied by v_mfma_scale_f32_16x16x128_f8f6f4.
//
// One workgroup per CU (or two) walks a list of BM x BN output tiles.  A stage
// is two K tiles (256 values of K) of both operands; NS ring slots, so NS - 1
// stages are in flight.  The loads go straight to LDS (lane l's 16 bytes land
// at 16 l of a tile, which is its operand), issued by asm with explicit waits:
// every wave issues the same number of loads in every stage (past the last
// stage, and in a stage without a scale piece, loads from an empty resource
// into a spare KiB), so a wait for all but the newest n is exact.  The scales
// come in pieces of four K tiles, with every other stage, into a ring of their
// own; a stage reads its two bytes per lane as one 16-bit LDS read.
#include <type_traits>

#include "mxfp4_device.h"

using namespace nh;

namespace {

template <int BM, int BN, int WGM, int WGN, int NS>
__device__ __forceinline__ void mx_gemm(const MxGemmArgs& a, int8_t* smem) {
    constexpr int NW = WGM * WGN, TA = BM / 16, TB = BN / 16, TT = TA + TB;
    constexpr int FM = TA / WGM, FN = TB / WGN;
    constexpr int LPW = (2 * TT + NW - 1) / NW;       // code loads per wave and stage
    constexpr int SPW = (TT / 4 + NW - 1) / NW;       // scale loads per wave and stage
    constexpr int kStage = 2 * TT * 1024, kPiece = TT * 256;
    constexpr int NP = NS;                            // scale pieces that the stages in flight span (K <= 256: one each)
    static_assert(TT % 4 == 0 && TA % WGM == 0 && TB % WGN == 0, "whole fragments");
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int wm = wave / WGN, wn = wave % WGN;
    const int KT = a.kt, KT2 = (KT + 1) >> 1;
    const int mtiles = (a.M + 15) >> 4, ntiles = (a.N + 15) >> 4;
    const uint32_t region = (uint32_t)KT * 1024u + (uint32_t)a.kq * 256u;
    const int tiles = a.tiles_m * a.tiles_n, G = gridDim.x, b = blockIdx.x;
    const int pos = (G & 7) == 0 ? (b & 7) * (G >> 3) + (b >> 3) : b;  // an XCD's workgroups side by side
    const int my_tiles = pos < tiles ? (tiles - 1 - pos) / G + 1 : 0;
    const int nst = my_tiles * KT2;
    if (nst == 0) return;
    typedef __attribute__((address_space(3))) int8_t lds_i8;
    const uint32_t ring = (uint32_t)(uintptr_t)(lds_i8*)smem;
    const uint32_t pieces = ring + (uint32_t)(NS * kStage);
    const uint32_t spare = pieces + (uint32_t)(NP * kPiece);
    const v4i none = rsrc_words(a.a, 0u);

    int it = 0, ik = 0, slot = 0, piece = 0;  // the next stage to issue
    v4i ra = none, rb = none;
    auto set_tile = [&]() {
        const int p = it * G + pos, mt0 = (p % a.tiles_m) * TA, nt0 = (p / a.tiles_m) * TB;
        ra = rsrc_words(a.a + (int64_t)mt0 * region, (uint32_t)min(TA, mtiles - mt0) * region);
        rb = rsrc_words(a.w + (int64_t)nt0 * region, (uint32_t)min(TB, ntiles - nt0) * region);
    };
    set_tile();
    auto issue = [&]() {
        const bool live = it < my_tiles;
        const uint32_t st = ring + (uint32_t)(slot * kStage);
#pragma unroll
        for (int i = 0; i < LPW; ++i) {
            const int q = wave + i * NW;  // uniform: [K half][A tiles, B tiles]
            const int h = q >= TT ? 1 : 0, t = q - h * TT, kt = 2 * ik + h;
            const bool ok = live && q < 2 * TT;
            const uint32_t off = kt < KT ? (uint32_t)(t < TA ? t : t - TA) * region + (uint32_t)(kt * 1024 + lane * 16)
                                         : (uint32_t)kOutOfRange;
            lds_dma16(!ok ? none : t < TA ? ra : rb, off, ok ? st + (uint32_t)(q * 1024) : spare);
        }
        const bool sc = live && (ik & 1) == 0;
#pragma unroll
        for (int i = 0; i < SPW; ++i) {
            const int q = wave + i * NW;  // four tiles' scale pieces
            const bool ok = sc && q < TT / 4;
            const int t = 4 * q;
            const uint32_t tile = (uint32_t)((t < TA ? t : t - TA) + (lane >> 4));
            const uint32_t off = tile * region + (uint32_t)(KT * 1024 + (ik >> 1) * 256 + (lane & 15) * 16);
            lds_dma16(!ok ? none : t < TA ? ra : rb, off, ok ? pieces + (uint32_t)(piece * kPiece + q * 1024) : spare);
        }
        if (live) {
            slot = slot + 1 == NS ? 0 : slot + 1;
            ++ik;
            if ((ik & 1) == 0 || ik == KT2) piece = piece + 1 == NP ? 0 : piece + 1;
            if (ik == KT2) {
                ik = 0;
                if (++it < my_tiles) set_tile();
            }
        }
    };
    static_assert(TA % 4 == 0, "a scale load is of one operand");

    v4f acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    int et = 0, rslot = 0, rpiece = 0, rk = 0;
    auto epilogue = [&]() {
        const int p = et * G + pos;
        const int m0 = (p % a.tiles_m) * BM + wm * FM * 16 + (lane & 15);
        const int n0 = (p / a.tiles_m) * BN + wn * FN * 16 + 4 * (lane >> 4);
        const bool bf16 = a.out_dtype == DT_BF16;
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            const int n = n0 + 16 * j;
            float bv[4] = {0.f, 0.f, 0.f, 0.f};
            if (a.bias)
#pragma unroll
                for (int r = 0; r < 4; ++r) bv[r] = n + r < a.N ? a.bias[n + r] : 0.0f;
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                const int m = m0 + 16 * i;
                float y[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) y[r] = a.bias ? acc[i][j][r] + bv[r] : acc[i][j][r];
                acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
                if (m >= a.M) continue;
                const int64_t o = (int64_t)m * a.N + n;
                if (n + 3 < a.N)
                    store_cols4((int8_t*)a.out + o * (bf16 ? 2 : 4), y, bf16);
                else
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (n + r < a.N) store_out(a.out, o + r, y[r], a.out_dtype);
            }
        }
        ++et;
    };
#pragma unroll
    for (int s = 0; s < NS - 1; ++s) issue();
    for (int g = 0; g < nst; ++g) {
        // stage g is in when all but the NS - 2 stages issued after it are
        wait_lgkm0();
        NH_WAIT_VMCNT((NS - 2) * (LPW + SPW));
        lds_barrier();
        issue();  // into the slot read last: every wave is past it
        const int8_t* st = smem + rslot * kStage + lane * 16;
        const uint8_t* sc = (const uint8_t*)smem + NS * kStage + rpiece * kPiece + lane * 4 + (rk & 1) * 2;
        int sa[FM], sb[FN];
#pragma unroll
        for (int i = 0; i < FM; ++i) sa[i] = *(const uint16_t*)(sc + (wm * FM + i) * 256);
#pragma unroll
        for (int j = 0; j < FN; ++j) sb[j] = *(const uint16_t*)(sc + (TA + wn * FN + j) * 256);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            v4i fa[FM], fb[FN];
#pragma unroll
            for (int i = 0; i < FM; ++i) fa[i] = *(const v4i*)(st + (h * TT + wm * FM + i) * 1024);
#pragma unroll
            for (int j = 0; j < FN; ++j) fb[j] = *(const v4i*)(st + (h * TT + TA + wn * FN + j) * 1024);
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int i = 0; i < FM; ++i)
                    acc[i][j] = h == 0 ? mx_mfma<0, 0>(fb[j], fa[i], acc[i][j], sb[j], sa[i])
                                       : mx_mfma<1, 1>(fb[j], fa[i], acc[i][j], sb[j], sa[i]);
        }
        rslot = rslot + 1 == NS ? 0 : rslot + 1;
        ++rk;
        if ((rk & 1) == 0 || rk == KT2) rpiece = rpiece + 1 == NP ? 0 : rpiece + 1;
        if (rk == KT2) {
            rk = 0;
            epilogue();
        }
    }
    NH_WAIT_VMCNT(0);  // the loads past the last stage write the spare KiB
}

}  // namespace

#define NH_MX_GEMM(name, BM, BN, WGM, WGN, NS, PER_SIMD)                                          \
    extern "C" __global__ __launch_bounds__(64 * WGM * WGN, PER_SIMD) void name(MxGemmArgs a) {   \
        extern __shared__ __align__(1024) int8_t smem[];                                          \
        mx_gemm<BM, BN, WGM, WGN, NS>(a, smem);                                                   \
    }
NH_MX_GEMM(nh_mx_gemm_256x256_kernel, 256, 256, 2, 4, 2, 2)
NH_MX_GEMM(nh_mx_gemm_128x128_kernel, 128, 128, 2, 2, 2, 2)
NH_MX_GEMM(nh_mx_gemm_64x64_kernel, 64, 64, 2, 2, 4, 2)
