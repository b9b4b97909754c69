// MXFP4 product of many rows: both operands in the tiled form, streamed into an
// LDS ring and multiplied by v_mfma_scale_f32_16x16x128_f8f6f4.
//
// A workgroup of WGM x WGN waves walks a list of BM x BN output tiles; a wave
// owns (BM / WGM) x (BN / WGN) of each.  A stage is KS K tiles (128 values of K
// each) of both operands; NS ring slots, NS - 1 stages in flight.
//  * The loads go straight to LDS (lane l's 16 bytes land at 16 l of a tile,
//    which is its operand).  They are asm with explicit waits: the compiler
//    would wait for all of them before each LDS read.  Every wave issues the
//    same number in every step, so a wait for all but the newest n is exact.
//    Past the last stage, past K and where a stage starts no piece of scales
//    they are of nothing (an offset or resource out of range): no branch in the
//    loop.
//  * Scales come in pieces of four K tiles, with the stage that starts one,
//    into a ring of their own, and are held as one dword per fragment.
//  * Tiles are dealt so that an XCD's workgroups hold neighbours of a
//    column-major order over the row tiles: they share weight panels in its L2.
// 2048 x 4096 -> 21504 takes 107 to 113 us by card, 7 of them the rows'
// quantization: 3.2 to 3.4 PFLOP/s.  The MFMAs alone, the CUs' load path and the
// LDS reads take about 50 us each and overlap in part: without loads 93 of 113,
// without seven of eight MFMAs 89, without the outputs' stores 96.  300 x
// 2701 -> 4099, 325 tiles of 64 x 64, takes 11: two or fewer workgroups per CU
// wait for each stage's loads.  So does a long K over few tiles: 1 x 21504 -> 4096,
// 64 of them, takes 30 us where its weights are 9.
#include "mxfp4_device.h"

using namespace nh;

namespace {

// A choice between values (between two variables it would be one of addresses,
// and put both in memory).
__device__ __forceinline__ v4i pick(bool c, v4i a, v4i b) {
    return v4i{c ? a[0] : b[0], c ? a[1] : b[1], c ? a[2] : b[2], c ? a[3] : b[3]};
}

// Scale pieces that NS stages can span: a piece is one stage of four K tiles,
// else two stages or more but for a tile's last, and a tile has two or more.
constexpr int mx_gemm_pieces(int ks, int ns) { return ks == 4 ? ns : ns / 2 + 1; }

template <int BM, int BN, int WGM, int WGN, int KS, int NS>
__device__ __forceinline__ void mx_gemm(const MxGemmArgs& a, int8_t* smem) {
    constexpr int NW = WGM * WGN, TA = BM / 16, TB = BN / 16, FM = TA / WGM, FN = TB / WGN;
    constexpr int LA = KS * TA / NW, LB = KS * TB / NW;    // code loads per wave and stage
    constexpr int SA = TA / 4, SB = TB / 4;                // scale loads per piece
    constexpr int SPW = (SA + SB + NW - 1) / NW;
    constexpr int LPW = LA + LB + SPW;                     // loads per wave and stage
    constexpr int kStage = KS * (TA + TB) * 1024, kPiece = (SA + SB) * 1024;
    constexpr int NP = mx_gemm_pieces(KS, NS);
    static_assert(KS * TA % NW == 0 && KS * TB % NW == 0 && TA % 4 == 0 && TB % 4 == 0, "a load is of one operand");
    static_assert(KS == 1 || KS == 2 || KS == 4, "a stage lies in one piece of scales");
    static_assert((NS - 2) * LPW < 64, "the wait's count");
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int wm = wave / WGN, wn = wave % WGN;
    const int KT = a.kt, KE = max(2, (KT + KS - 1) / KS);  // stages per tile (of nothing past K)
    const int mtiles = (a.M + 15) >> 4, ntiles = (a.N + 15) >> 4;
    const uint32_t region = (uint32_t)KT * 1024u + (uint32_t)a.kq * 256u;
    const int tiles = a.tiles_m * a.tiles_n, G = gridDim.x, b = blockIdx.x;
    const int pos = (G & 7) == 0 ? (b & 7) * (G >> 3) + (b >> 3) : b;
    const int my_tiles = pos < tiles ? (tiles - 1 - pos) / G + 1 : 0;
    if (my_tiles == 0) return;
    typedef __attribute__((address_space(3))) int8_t lds_i8;
    const uint32_t ring = (uint32_t)(uintptr_t)(lds_i8*)smem;
    const uint32_t pieces = ring + (uint32_t)(NS * kStage);
    const uint32_t spare = pieces + (uint32_t)(NP * kPiece);
    const uint32_t vlane = (uint32_t)lane * 16u;
    const uint32_t vscale = (uint32_t)(lane >> 4) * region + (uint32_t)KT * 1024u + (uint32_t)(lane & 15) * 16u;

    // the next stage to issue
    int it = -1, ik = 0, islot = 0, ipiece = 0;
    const v4i none = rsrc_words(a.a, 0u);
    v4i ra, rb, pa, pb;  // the tile's operands, and the next tile's
    auto set_next = [&]() {
        const int p = (it + 1) * G + pos, mt0 = (p % a.tiles_m) * TA, nt0 = (p / a.tiles_m) * TB;
        const bool live = it + 1 < my_tiles;
        pa = rsrc_words(a.a + (int64_t)mt0 * region, live ? (uint32_t)min(TA, mtiles - mt0) * region : 0u);
        pb = rsrc_words(a.w + (int64_t)nt0 * region, live ? (uint32_t)min(TB, ntiles - nt0) * region : 0u);
    };
    set_next();
    ra = pa;
    rb = pb;
    it = 0;
    set_next();
    bool wrapped = false;
    auto issue = [&]() {
        const uint32_t st = ring + (uint32_t)(islot * kStage);
#pragma unroll
        for (int i = 0; i < LA + LB; ++i) {
            // A [KS][TA], then B [KS][TB]; a wave's i-th is of one operand
            const bool of_a = i < LA;
            const int n = of_a ? TA : TB, q = wave + (of_a ? i : i - LA) * NW, h = q / n, t = q - h * n, kt = ik * KS + h;
            const uint32_t k = kt < KT ? (uint32_t)kt * 1024u : (uint32_t)kOutOfRange - 16u * region;
            lds_dma16(pick(of_a, ra, rb), vlane + ((uint32_t)t * region + k),
                      st + (uint32_t)(((of_a ? 0 : KS * TA) + q) * 1024));
        }
        const bool piece = (ik * KS & 3) == 0;
#pragma unroll
        for (int i = 0; i < SPW; ++i) {  // four tiles' pieces
            const int q = wave + i * NW;
            const bool live = piece && q < SA + SB, of_a = q < SA;
            const uint32_t off = (uint32_t)(4 * (of_a ? q : q - SA)) * region + (uint32_t)(ik * KS >> 2) * 256u;
            lds_dma16(pick(live && ik * KS < KT, pick(of_a, ra, rb), none), vscale + off,
                      live ? pieces + (uint32_t)(ipiece * kPiece + q * 1024) : spare);
        }
        islot = islot + 1 == NS ? 0 : islot + 1;
        ++ik;
        const bool wrap = ik == KE;
        ipiece = (ik * KS & 3) == 0 || wrap ? (ipiece + 1 == NP ? 0 : ipiece + 1) : ipiece;
        ik = wrap ? 0 : ik;
        it += wrap ? 1 : 0;
        ra = pick(wrap, pa, ra);
        rb = pick(wrap, pb, rb);
        wrapped = wrap;
    };

    v4f acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    // Output of the tile: whole tiles in bf16 with 16-byte stores.  Lane 16 g + m
    // has columns 4 g .. 4 g + 3 of row m of fragments j and j + 1; swapping odd
    // lane rows of the one with even lane rows of the other leaves eight
    // consecutive columns in each lane, and 64 bytes of a row in four lanes.
    int et = 0;
    auto epilogue = [&]() {
        const int p = et * G + pos;
        const int mt = (p % a.tiles_m) * BM, nt = (p / a.tiles_m) * BN;
        const int m0 = mt + wm * FM * 16 + (lane & 15), n0 = nt + wn * FN * 16;
        const bool bf16 = a.out_dtype == DT_BF16;
        ++et;
        if (bf16 && mt + BM <= a.M && nt + BN <= a.N && FN % 2 == 0) {
            const int g = lane >> 4;
            uint16_t* row = (uint16_t*)a.out + (int64_t)m0 * a.N + n0 + (g & 1) * 16 + (g >> 1) * 8;
            float bv[FN][4];
            if (a.bias)
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) bv[j][r] = a.bias[n0 + j * 16 + 4 * g + r];
#pragma unroll
            for (int i = 0; i < FM; ++i) {
#pragma unroll
                for (int j = 0; j < FN; j += 2) {
                    uint32_t w[4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float y[4];
#pragma unroll
                        for (int r = 0; r < 4; ++r) y[r] = acc[i][j + h][r];
                        if (a.bias) {
#pragma unroll
                            for (int r = 0; r < 4; ++r) y[r] = y[r] + bv[j + h][r];
                        }
                        w[2 * h] = f32x2_to_bf16x2(y[0], y[1]);
                        w[2 * h + 1] = f32x2_to_bf16x2(y[2], y[3]);
                        acc[i][j + h] = v4f{0.f, 0.f, 0.f, 0.f};
                    }
                    const auto lo = __builtin_amdgcn_permlane16_swap(w[0], w[2], false, false);
                    const auto hi = __builtin_amdgcn_permlane16_swap(w[1], w[3], false, false);
                    const uint32_t v[4] = {lo[0], hi[0], lo[1], hi[1]};
                    __builtin_memcpy(row + j * 16, v, 16);
                }
                row += (int64_t)16 * a.N;
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            const int n = n0 + 16 * j + 4 * (lane >> 4);
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
    };

#pragma unroll
    for (int s = 0; s < NS - 1; ++s) {
        issue();
        if (wrapped) set_next();
    }
    int rslot = 0, rpiece = 0, rk = 0;
    int ca[FM], cb[FN];
    for (int t = 0; t < my_tiles; ++t) {
        for (int k = 0; k < KE; ++k) {
            // the stage is in when all but the NS - 2 behind it are, and the slot
            // of the one before it free when every wave is here
            wait_lgkm0();
            NH_WAIT_VMCNT((NS - 2) * LPW);
            lds_barrier();
            // scale dwords of the piece, a byte of them per K tile
            if ((rk * KS & 3) == 0) {
                const uint8_t* sc = (const uint8_t*)smem + NS * kStage + rpiece * kPiece + lane * 4;
#pragma unroll
                for (int j = 0; j < FN; ++j) cb[j] = *(const int*)(sc + (TA + wn * FN + j) * 256);
#pragma unroll
                for (int i = 0; i < FM; ++i) ca[i] = *(const int*)(sc + (wm * FM + i) * 256);
            }
            v4i fa[KS][FM], fb[KS][FN];
            const int8_t* st = smem + rslot * kStage + lane * 16;
#pragma unroll
            for (int h = 0; h < KS; ++h) {
#pragma unroll
                for (int j = 0; j < FN; ++j) fb[h][j] = *(const v4i*)(st + (KS * TA + h * TB + wn * FN + j) * 1024);
#pragma unroll
                for (int i = 0; i < FM; ++i) fa[h][i] = *(const v4i*)(st + (h * TA + wm * FM + i) * 1024);
            }
            issue();
#pragma unroll
            for (int h = 0; h < KS; ++h)
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int i = 0; i < FM; ++i) {
                        if (h == 0) acc[i][j] = mx_mfma<0, 0>(fb[h][j], fa[h][i], acc[i][j], cb[j], ca[i]);
                        if (h == 1) acc[i][j] = mx_mfma<1, 1>(fb[h][j], fa[h][i], acc[i][j], cb[j], ca[i]);
                        if (h == 2) acc[i][j] = mx_mfma<2, 2>(fb[h][j], fa[h][i], acc[i][j], cb[j], ca[i]);
                        if (h == 3) acc[i][j] = mx_mfma<3, 3>(fb[h][j], fa[h][i], acc[i][j], cb[j], ca[i]);
                    }
            if constexpr (KS < 4) {
#pragma unroll
                for (int j = 0; j < FN; ++j) cb[j] = (int)((uint32_t)cb[j] >> (8 * KS));
#pragma unroll
                for (int i = 0; i < FM; ++i) ca[i] = (int)((uint32_t)ca[i] >> (8 * KS));
            }
            if (wrapped) set_next();
            ++rk;
            const bool wrap = rk == KE;
            rslot = rslot + 1 == NS ? 0 : rslot + 1;
            rpiece = (rk * KS & 3) == 0 || wrap ? (rpiece + 1 == NP ? 0 : rpiece + 1) : rpiece;
            rk = wrap ? 0 : rk;
        }
        epilogue();
    }
    NH_WAIT_VMCNT(0);  // the loads of nothing behind the last stage
}

}  // namespace

#define NH_MX_GEMM(name, BM, BN, WGM, WGN, KS, NS)                                            \
    extern "C" __global__ __launch_bounds__(64 * WGM * WGN, 2) void name(MxGemmArgs a) {      \
        extern __shared__ __align__(1024) int8_t smem[];                                      \
        mx_gemm<BM, BN, WGM, WGN, KS, NS>(a, smem);                                           \
    }
NH_MX_GEMM(nh_mx_gemm_256x256_kernel, 256, 256, 2, 4, 1, 4)
NH_MX_GEMM(nh_mx_gemm_128x128_kernel, 128, 128, 2, 2, 1, 4)
NH_MX_GEMM(nh_mx_gemm_64x64_kernel, 64, 64, 2, 2, 4, 2)
