// Low-rank adapters of many requests beside a linear layer, and their gradients.
//
// Row i belongs to adapter l (or to none); A_l [r][k], B_l [n][r], s_l:
//   h_i = A_l x_i,   out_i = base_i + s_l B_l h_i
//   dh_i = s_l B_l^T dout_i,   dx_i = dx_base_i + A_l^T dh_i,
//   dA_l = sum_i dh_i x_i^T,   dB_l = sum_i dout_i (s_l h_i)^T.
// Three products make them all, over rows gathered by adapter:
//   shrink: rows x matrix, summed over a long axis C (x A^T, dout B), in parts;
//   expand: low-rank values x matrix, added to rows of length C (h B^T, dh A);
//   outer:  columns of rows x low-rank values, summed over rows (dA, dB).
// Low-rank values stay in f32.  Where both operands come as bf16 the products
// run on the bf16 matrix cores: an f32 low-rank value is cut into three bf16
// parts of eight significant bits each (by truncation, so v = hi + mid + lo
// exactly while lo is normal), whose products with bf16 are exact in the f32
// sums; bf16 results take the first two parts (off by 2^-16 of a term, 2^-7 of
// the result's own rounding).  Otherwise the f32 matrix cores take every value as
// it is.  Every sum has a fixed order: results do not change from run to run.
//
// A row's products see its own values only; what stands in rows without an
// adapter, or in another adapter's matrices, reaches no other row.
#include "nh_device.h"

using namespace nh;

namespace {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

constexpr int kTileRows = 64;  // slots per tile of the plan

// ---- operands of a matrix instruction: eight values per lane, of lane l for row
// or column l % 16 and K 8 (l / 16) .. + 7
struct Frag16 {
    static constexpr bool bf16 = true;
    v4i v;
};
struct Frag32 {
    static constexpr bool bf16 = false;
    float v[8];
};

__device__ __forceinline__ void clear(Frag16& f) { f.v = v4i{0, 0, 0, 0}; }
__device__ __forceinline__ void clear(Frag32& f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f.v[i] = 0.0f;
}

// Eight consecutive values.
__device__ __forceinline__ void load8(const void* p, int64_t at, int dtype, Frag16& f) {
    __builtin_memcpy(&f.v, (const uint16_t*)p + at, 16);
}
__device__ __forceinline__ void load8(const void* p, int64_t at, int dtype, Frag32& f) {
    if (dtype == DT_BF16) {
        v4i h;
        __builtin_memcpy(&h, (const uint16_t*)p + at, 16);
        unpack_bf16x8(h, f.v);
    } else {
        __builtin_memcpy(f.v, (const float*)p + at, 32);
    }
}

// Eight values `stride` apart, the first `n` of them there, zeros behind.
__device__ __forceinline__ void load8(const void* p, int64_t at, int64_t stride, int dtype, int n, Frag16& f) {
    const uint16_t* q = (const uint16_t*)p + at;
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = i < n ? q[i * stride] : 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) f.v[i] = (int)(u[2 * i] | (u[2 * i + 1] << 16));
}
__device__ __forceinline__ void load8(const void* p, int64_t at, int64_t stride, int dtype, int n, Frag32& f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f.v[i] = i < n ? load_as_f32(p, at + i * stride, dtype) : 0.0f;
}

// acc += a b over 32 K: rows of a down the lane's four, b's columns by lane.
__device__ __forceinline__ v4f mma(const Frag16& a, const Frag16& b, v4f acc) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a.v), __builtin_bit_cast(v8bf, b.v), acc, 0, 0, 0);
}
__device__ __forceinline__ v4f mma(const Frag32& a, const Frag32& b, v4f acc) {
#pragma unroll
    for (int i = 0; i < 8; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], acc, 0, 0, 0);
    return acc;
}

// A block of bf16 rows in LDS, `pitch` values from one to the next, as operands
// whose K runs down the rows: lane l gets rows 8 (l / 16) .. + 7 of column
// col(l % 16).  A transposing read gives each of 16 lanes four rows of its column,
// lane l having addressed row l / 4 of them, columns col(4 (l % 4)) .. + 3.
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

template <class Col>
__device__ __forceinline__ void load_rows(const uint16_t* lds, int pitch, Col col, Frag16& f) {
    const int lane = threadIdx.x & 63, l16 = lane & 15, row = 8 * (lane >> 4) + (l16 >> 2), c = col(4 * (l16 & 3));
    const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(lds + row * pitch + c));
    const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(lds + (row + 4) * pitch + c));
    const uint64_t u[2] = {__builtin_bit_cast(uint64_t, lo), __builtin_bit_cast(uint64_t, hi)};
    f.v = v4i{(int)u[0], (int)(u[0] >> 32), (int)u[1], (int)(u[1] >> 32)};
}

// What a wave wrote to its own part of LDS is there for its own reads.
__device__ __forceinline__ void wave_lds_sync() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14));  // lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// Eight f32 values as an operand: PARTS bf16 parts, or as they are.  A value
// that is not finite is its first part, with zeros behind.
template <int PARTS>
struct Split16 {
    static constexpr int parts = PARTS;
    Frag16 f[PARTS];
};
struct Split32 {
    static constexpr int parts = 1;
    Frag32 f[1];
};

__device__ __forceinline__ uint32_t bf16_part(float& v) {
    const uint32_t u = f32_bits(v);
    if ((u & 0x7f800000u) == 0x7f800000u) {
        v = 0.0f;
        return (u >> 16) | ((u & 0x7fffffu) ? 0x40u : 0u);
    }
    v = v - f32_from_bits(u & 0xffff0000u);  // exact
    return u >> 16;
}

template <int PARTS>
__device__ __forceinline__ void split8(const float (&v)[8], Split16<PARTS>& s) {
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = v[i];
#pragma unroll
    for (int q = 0; q < PARTS; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t lo = bf16_part(r[2 * i]), hi = bf16_part(r[2 * i + 1]);
            s.f[q].v[i] = (int)(lo | (hi << 16));
        }
}
__device__ __forceinline__ void split8(const float (&v)[8], Split32& s) {
#pragma unroll
    for (int i = 0; i < 8; ++i) s.f[0].v[i] = v[i];
}

// ---- the rows of a workgroup ---------------------------------------------------
// Tile `tile`: its adapter (`adapters`: rows without one) and its rows; returns how
// many (0: nothing to do), uniform.  64 at a time from the plan, or (FEW) 16 of at
// most 64 rows in all, where every row that is the 1st, 17th, .. of its adapter
// leads a tile.
template <bool FEW>
__device__ __forceinline__ int lora_tile(const LoraArgs& a, int tile, int* rows, int& adapter) {
    const int lane = threadIdx.x & 63;
    if constexpr (FEW) {
        int e = -1;
        if (lane < a.m) {
            e = a.ids[lane];
            if (e < 0 || e >= a.adapters) e = a.adapters;
        }
        adapter = __builtin_amdgcn_readlane(e, tile);
        const uint64_t same = __ballot(e == adapter);
        const int before = __popcll(same & ((1ull << tile) - 1));
        if (before % 16 != 0) return 0;  // uniform
        const int mine = __popcll(same & ((1ull << lane) - 1)) - before;
        if (threadIdx.x < 64 && e == adapter && mine >= 0 && mine < 16) rows[mine] = lane;
        __syncthreads();
        return min(16, __popcll(same) - before);
    } else {
        if (tile >= a.counts[0]) return 0;
        adapter = a.tile_adapter[tile];
        const int row = a.slot_row[(int64_t)tile * kTileRows + lane];  // those without a row are the last
        if (threadIdx.x < 64) rows[lane] = row;
        __syncthreads();
        return __popcll(__ballot(row >= 0));
    }
}

// ---- shrink --------------------------------------------------------------------
// part[split][row][rank] = sum over the split's columns of x[row][c] w(rank, c).
// The waves of a workgroup take consecutive parts of the columns, each for all of
// the tile's rows, so that a matrix is read once per tile, and add up through LDS.
// Ranks past the last and rows past the tile's are computed on the nearest valid
// operand and not read again; columns past C are zeros in both operands.
// A matrix of [C][rank] (COLS) goes through LDS, 32 of its rows at a time.
template <class Frag, bool FEW, int RT, bool COLS>
__device__ __forceinline__ void lora_shrink(const LoraArgs& a) {
    constexpr int RB = FEW ? 1 : 4, RP = 16 * RT, kPlane = 256 * RB * RT;
    extern __shared__ float lora_lds[];  // half the waves' sums; before: a wave's 32 rows of a [C][rank] matrix each
    __shared__ int rows[16 * RB];
    int adapter;
    const int count = lora_tile<FEW>(a, blockIdx.x, rows, adapter);
    if (count == 0 || adapter == a.adapters) return;  // uniform
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = blockDim.x >> 7, g = lane >> 4, l16 = lane & 15;
    const int64_t first = ((int64_t)blockIdx.y * (blockDim.x >> 6) + wave) * a.per_wave;
    const int c0 = (int)min((int64_t)a.C, first), c1 = min(a.C, c0 + a.per_wave);
    int64_t xat[RB], wat[RT];
#pragma unroll
    for (int b = 0; b < RB; ++b) xat[b] = (int64_t)rows[min(16 * b + l16, count - 1)] * a.C;
    const int64_t matrix = (int64_t)adapter * a.rank * a.C;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int rank = min(16 * r + l16, a.rank - 1);
        wat[r] = matrix + (COLS ? rank : (int64_t)rank * a.C);
    }
    v4f acc[RB][RT];
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int r = 0; r < RT; ++r) acc[b][r] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    constexpr bool staged = COLS && Frag::bf16;
    uint16_t* block = (uint16_t*)lora_lds + wave * 32 * RP;
    // 32 columns from c on: operands, of which the last may be past the end
    auto load_x = [&](int c, Frag (&x)[RB]) {
        const int at = c + 8 * g;
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            if (16 * b >= count) continue;  // uniform
            if (at + 8 <= a.C) load8(a.x, xat[b] + at, a.x_dtype, x[b]);
            else load8(a.x, xat[b] + at, 1, a.x_dtype, a.C - at, x[b]);
        }
    };
    auto load_w = [&](int c, Frag (&w)[RT]) {
        if constexpr (staged) {
            // rows c .. c + 31 of the matrix, zeros past C; ranks past the last are not read again
            const int64_t from = matrix + (int64_t)c * a.rank;
            const int there = min(32, a.C - c);
            if (a.rank % 8 == 0) {
                const int vectors = a.rank >> 3;  // per row
                for (int i = lane; i < 32 * vectors; i += 64) {
                    const int row = i / vectors;
                    Frag16 v;
                    clear(v);
                    if (row < there) load8(a.w, from + 8 * i, DT_BF16, v);
                    *(v4i*)(block + row * RP + 8 * (i - row * vectors)) = v.v;
                }
            } else {
                for (int i = lane; i < 32 * a.rank; i += 64) {
                    const int row = i / a.rank;
                    block[row * RP + i - row * a.rank] = row < there ? ((const uint16_t*)a.w)[from + i] : 0;
                }
            }
            wave_lds_sync();
#pragma unroll
            for (int r = 0; r < RT; ++r) load_rows(block, RP, [&](int i) { return 16 * r + i; }, w[r]);
        } else {
            const int at = c + 8 * g;
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                if constexpr (COLS) {
                    load8(a.w, wat[r] + (int64_t)at * a.rank, a.rank, a.w_dtype, a.C - at, w[r]);
                } else {
                    if (at + 8 <= a.C) load8(a.w, wat[r] + at, a.w_dtype, w[r]);
                    else load8(a.w, wat[r] + at, 1, a.w_dtype, a.C - at, w[r]);
                }
            }
        }
    };
    constexpr int UN = staged || RT == 8 || !Frag::bf16 ? 1 : FEW ? 4 : 2;
    for (int c = c0; c < c1; c += 32 * UN) {
        Frag x[UN][RB], w[UN][RT];
#pragma unroll
        for (int u = 0; u < UN; ++u)
            if (c + 32 * u < c1) {
                load_x(c + 32 * u, x[u]);
                load_w(c + 32 * u, w[u]);
            }
#pragma unroll
        for (int u = 0; u < UN; ++u)
            if (c + 32 * u < c1) {
#pragma unroll
                for (int b = 0; b < RB; ++b)
                    if (16 * b < count) {
#pragma unroll
                        for (int r = 0; r < RT; ++r) acc[b][r] = mma(w[u][r], x[u][b], acc[b][r]);
                    }
            }
    }
    // the waves' sums: the second half's, the first half's onto them, then all in order
    if (staged) __syncthreads();
    float* mine = lora_lds + (wave % half) * kPlane + l16 * RP + 4 * g;
    for (int turn = 0; turn < 2; ++turn) {
        if ((wave >= half) == (turn == 0)) {
#pragma unroll
            for (int b = 0; b < RB; ++b)
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    v4f* p = (v4f*)(mine + 16 * b * RP + 16 * r);
                    *p = turn == 0 ? acc[b][r] : acc[b][r] + *p;
                }
        }
        __syncthreads();
    }
    for (int i = 4 * threadIdx.x; i < count * RP; i += 4 * blockDim.x) {
        v4f v = *(v4f*)(lora_lds + i);
        for (int w = 1; w < half; ++w) v += *(v4f*)(lora_lds + w * kPlane + i);
        *(v4f*)(a.part + ((int64_t)blockIdx.y * a.m + rows[i / RP]) * RP + i % RP) = v;
    }
}

// ---- expand --------------------------------------------------------------------
// out[row][c] = base[row][c] + sum over ranks of (s) h[row][rank] w(rank, c), h the
// sum of shrink's parts in order.  A wave has 16 rows (of a plan's tile each of the
// four its own, of a few rows all the same and every fourth step of the columns)
// and 64 columns a step: four tiles, those of a pair interleaved by fours, so that
// a lane's results are eight consecutive ones.  A matrix of [rank][C] goes through
// LDS, a wave's step at a time.
template <class Frag, class Split, bool FEW, int RT, bool COLS>
__device__ __forceinline__ void lora_expand_columns(const LoraArgs& a, const int* rows, int count, int adapter,
                                                    uint16_t* block) {
    constexpr int KC = (RT + 1) / 2, RP = 16 * RT;  // steps of 32 ranks
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, l16 = lane & 15;
    const int own = FEW ? 0 : 16 * wave;
    if (own >= count) return;  // uniform in the wave
    const int c0 = (int)min((int64_t)a.C, (int64_t)blockIdx.y * a.columns) + (FEW ? 64 * wave : 0);
    const int c1 = (int)min((int64_t)a.C, (int64_t)(blockIdx.y + 1) * a.columns);
    const int row = rows[min(own + l16, count - 1)];
    const bool mine = own + l16 < count;
    const int64_t at = (int64_t)row * a.C, matrix = (int64_t)adapter * a.rank * a.C;
    const bool whole = a.rank % 8 == 0;
    // the step's matrix operands
    auto load_w = [&](int c, Frag (&w)[4][KC]) {
        if constexpr (Frag::bf16 && !COLS) {
            // ranks by row, eight lanes each; ranks past the last and columns past C are zeros
#pragma unroll
            for (int r0 = 0; r0 < 32 * KC; r0 += 8) {
                const int rank = r0 + (lane >> 3), col = c + 8 * (lane & 7);
                Frag16 v;
                clear(v);
                if (rank < a.rank) {
                    const int64_t p = matrix + (int64_t)rank * a.C + col;
                    if (col + 8 <= a.C) load8(a.w, p, DT_BF16, v);
                    else load8(a.w, p, 1, DT_BF16, a.C - col, v);
                }
                *(v4i*)(block + rank * 64 + 8 * (lane & 7)) = v.v;
            }
            wave_lds_sync();
#pragma unroll
            for (int p = 0; p < 4; ++p)
#pragma unroll
                for (int q = 0; q < KC; ++q)
                    load_rows(block + 32 * q * 64, 64, [&](int i) { return 32 * (p >> 1) + 2 * i + 4 * (p & 1); }, w[p][q]);
        } else {
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const int col = min(c + 32 * (p >> 1) + 8 * (l16 >> 2) + 4 * (p & 1) + (l16 & 3), a.C - 1);
#pragma unroll
                for (int q = 0; q < KC; ++q) {
                    const int rank = 32 * q + 8 * g;
                    if constexpr (COLS) {
                        const int64_t from = matrix + (int64_t)col * a.rank + rank;
                        if (whole) {
                            if (rank < a.rank) load8(a.w, from, a.w_dtype, w[p][q]);
                            else clear(w[p][q]);
                        } else {
                            load8(a.w, from, 1, a.w_dtype, a.rank - rank, w[p][q]);
                        }
                    } else {
                        load8(a.w, matrix + (int64_t)rank * a.C + col, a.C, a.w_dtype, a.rank - rank, w[p][q]);
                    }
                }
            }
        }
    };
    const bool bf16_out = a.out_dtype == DT_BF16;
    auto load_base = [&](int c, Frag32 (&base)[2]) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const int first = c + 32 * p + 8 * g, there = a.C - first;
            clear(base[p]);
            if (!a.base || !mine || there <= 0) continue;
            if (there >= 8) load8(a.base, at + first, a.out_dtype, base[p]);
            else load8(a.base, at + first, 1, a.out_dtype, there, base[p]);
        }
    };
    // the low-rank values, while the first step's operands are on their way
    Frag w[4][KC];
    Frag32 base[2];
    if (c0 < c1) {
        load_w(c0, w);
        load_base(c0, base);
    }
    Split h[KC];
    const float scale = a.scaled && a.scales ? a.scales[adapter] : 1.0f;
#pragma unroll
    for (int q = 0; q < KC; ++q) {
        float v[8];
        const int rank = 32 * q + 8 * g;
        const float* p = a.part + (int64_t)row * RP + rank;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
        if (rank < RP) {
            for (int s = 0; s < a.splits; ++s) {
                float t[8];
                __builtin_memcpy(t, p + (int64_t)s * a.m * RP, 32);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = s == 0 ? t[i] : v[i] + t[i];
            }
        }
        const bool first = blockIdx.y == 0 && (!FEW || wave == 0) && a.h_out && mine;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (rank + i >= a.rank) v[i] = 0.0f;
            else if (first) a.h_out[(int64_t)row * a.rank + rank + i] = v[i];
            v[i] *= scale;
            if (rank + i >= a.rank) v[i] = 0.0f;  // a scale without a value
        }
        split8(v, h[q]);
    }
    constexpr int kStep = FEW ? 256 : 64;
    for (int c = c0; c < c1; c += kStep) {
        v4f acc[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            acc[p] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = Split::parts - 1; s >= 0; --s)  // the small parts first
#pragma unroll
                for (int q = 0; q < KC; ++q) acc[p] = mma(w[p][q], h[q].f[s], acc[p]);
        }
        float v[2][8];
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[p][i] = base[p].v[i] + acc[2 * p + (i >> 2)][i & 3];
        if (c + kStep < c1) {
            load_w(c + kStep, w);
            load_base(c + kStep, base);
        }
        if (!mine) continue;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const int first = c + 32 * p + 8 * g, there = a.C - first;
            if (there >= 8) {
                if (bf16_out) {
                    const uint32_t u[4] = {f32x2_to_bf16x2(v[p][0], v[p][1]), f32x2_to_bf16x2(v[p][2], v[p][3]),
                                           f32x2_to_bf16x2(v[p][4], v[p][5]), f32x2_to_bf16x2(v[p][6], v[p][7])};
                    __builtin_memcpy((uint16_t*)a.out + at + first, u, 16);
                } else {
                    __builtin_memcpy((float*)a.out + at + first, v[p], 32);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < there) store_out(a.out, at + first + i, v[p][i], a.out_dtype);
            }
        }
    }
}

template <class Frag, bool FEW, int RT, bool COLS>
__device__ __forceinline__ void lora_expand(const LoraArgs& a) {
    constexpr bool staged = Frag::bf16 && !COLS;
    __shared__ int rows[FEW ? 16 : kTileRows];
    __shared__ __align__(16) uint16_t blocks[staged ? 4 * 32 * ((RT + 1) / 2) * 64 : 8];
    int adapter;
    const int count = lora_tile<FEW>(a, blockIdx.x, rows, adapter);
    if (count == 0) return;  // uniform
    if (adapter == a.adapters) {  // rows without an adapter: the base
        const int start = (int)min((int64_t)a.C, (int64_t)blockIdx.y * a.columns);
        const int end = (int)min((int64_t)a.C, (int64_t)(blockIdx.y + 1) * a.columns);
        if (blockIdx.y == 0 && a.h_out)
            for (int i = threadIdx.x; i < count * a.rank; i += blockDim.x)
                a.h_out[(int64_t)rows[i / a.rank] * a.rank + i % a.rank] = 0.0f;
        if (a.base == a.out) return;
        for (int r = 0; r < count; ++r) {
            const int64_t at = (int64_t)rows[r] * a.C;
            for (int c = start + 8 * threadIdx.x; c < end; c += 8 * blockDim.x) {
                if (c + 8 <= end && a.base) {  // as they are
                    uint32_t u[8];
                    if (a.out_dtype == DT_BF16) {
                        __builtin_memcpy(u, (const uint16_t*)a.base + at + c, 16);
                        __builtin_memcpy((uint16_t*)a.out + at + c, u, 16);
                    } else {
                        __builtin_memcpy(u, (const float*)a.base + at + c, 32);
                        __builtin_memcpy((float*)a.out + at + c, u, 32);
                    }
                } else {
                    for (int i = c; i < min(c + 8, end); ++i)
                        store_out(a.out, at + i, a.base ? load_as_f32(a.base, at + i, a.out_dtype) : 0.0f, a.out_dtype);
                }
            }
        }
        return;
    }
    uint16_t* block = blocks + (staged ? (threadIdx.x >> 6) * 32 * ((RT + 1) / 2) * 64 : 0);
    if constexpr (!Frag::bf16)
        lora_expand_columns<Frag, Split32, FEW, RT, COLS>(a, rows, count, adapter, block);
    else if (a.out_dtype == DT_BF16)
        lora_expand_columns<Frag, Split16<2>, FEW, RT, COLS>(a, rows, count, adapter, block);
    else
        lora_expand_columns<Frag, Split16<3>, FEW, RT, COLS>(a, rows, count, adapter, block);
}

// ---- outer ---------------------------------------------------------------------
// grad(rank, c) of an adapter = sum over its rows of ht[rank][slot] x[row][c].  An
// item of the plan is some of an adapter's tiles; one that has them all writes the
// gradient, the others a partial sum each.  A wave has 64 columns, 32 rows a step,
// which bf16 takes through LDS; the next step's rows are on their way meanwhile.
template <class Frag, int RT, bool COLS>
__device__ __forceinline__ void lora_outer(const LoraArgs& a) {
    constexpr int PARTS = Frag::bf16 ? 3 : 1, CT = 4;
    __shared__ __align__(16) uint16_t blocks[Frag::bf16 ? 4 * 32 * 64 : 8];
    if ((int)blockIdx.y >= a.counts[1]) return;
    const int32_t* item = a.items + 4 * blockIdx.y;
    const int adapter = item[0], tile = item[1], tiles = item[2], partial = item[3];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, l16 = lane & 15;
    const int64_t first = ((int64_t)blockIdx.x * 4 + wave) * 16 * CT;
    if (first >= a.C) return;
    const int c0 = (int)first;
    v4f acc[CT][RT];
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int r = 0; r < RT; ++r) acc[c][r] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    const int64_t s0 = (int64_t)tile * kTileRows, s1 = s0 + (int64_t)tiles * kTileRows;
    uint16_t* block = blocks + (Frag::bf16 ? wave * 32 * 64 : 0);
    // bf16: a lane loads eight columns of four rows
    const int col8 = c0 + 8 * (lane & 7);
    v4i ahead[4];
    auto load_rows32 = [&](int64_t s) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = a.slot_row[s + 8 * i + (lane >> 3)];
            Frag16 v;
            clear(v);
            if (row >= 0) {
                const int64_t p = (int64_t)row * a.C + col8;
                if (col8 + 8 <= a.C) load8(a.x, p, DT_BF16, v);
                else load8(a.x, p, 1, DT_BF16, a.C - col8, v);
            }
            ahead[i] = v.v;
        }
    };
    if constexpr (Frag::bf16) load_rows32(s0);
    for (int64_t s = s0; s < s1; s += 32) {
        const int64_t at = s + 8 * g;
        Frag x[CT], h[RT][PARTS];
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
                load8(a.ht, ((int64_t)p * (16 * RT) + 16 * r + l16) * a.slots + at, DT_F32, h[r][p]);
        if constexpr (Frag::bf16) {
#pragma unroll
            for (int i = 0; i < 4; ++i) *(v4i*)(block + (8 * i + (lane >> 3)) * 64 + 8 * (lane & 7)) = ahead[i];
            wave_lds_sync();
#pragma unroll
            for (int c = 0; c < CT; ++c) load_rows(block, 64, [&](int i) { return 16 * c + i; }, x[c]);
            if (s + 32 < s1) load_rows32(s + 32);
        } else {
            int row[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) row[i] = a.slot_row[at + i];
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                const int col = min(c0 + 16 * c + l16, a.C - 1);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    x[c].v[i] = row[i] >= 0 ? load_as_f32(a.x, (int64_t)row[i] * a.C + col, a.x_dtype) : 0.0f;
            }
        }
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int p = PARTS - 1; p >= 0; --p)
                    acc[c][r] = COLS ? mma(h[r][p], x[c], acc[c][r]) : mma(x[c], h[r][p], acc[c][r]);
    }
    const bool add = partial < 0 && a.accumulate;
    float* to = partial < 0 ? a.grad + (int64_t)adapter * a.rank * a.C : a.gpart + (int64_t)partial * a.rank * a.C;
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            // COLS: the lane's column, four ranks; else the lane's rank, four columns
            const int col = c0 + 16 * c + (COLS ? l16 : 4 * g), rank = 16 * r + (COLS ? 4 * g : l16);
            if (col >= a.C || rank >= a.rank) continue;
            float* p = to + (COLS ? (int64_t)col * a.rank + rank : (int64_t)rank * a.C + col);
            const int there = COLS ? a.rank - rank : a.C - col;
            if (there >= 4) {
                v4f v = acc[c][r];
                if (add) {
                    v4f old;
                    __builtin_memcpy(&old, p, 16);
                    v += old;
                }
                __builtin_memcpy(p, &v, 16);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (i < there) p[i] = add ? p[i] + acc[c][r][i] : acc[c][r][i];
            }
        }
}

}  // namespace

// ---- the plan ------------------------------------------------------------------
// One workgroup sorts the rows by adapter, stable by row, rows without one last,
// each adapter's from a tile of its own on; the waves take consecutive parts of the
// rows.  A wave ranks 64 rows at a time among its rows of the same adapter by
// ballots, and keeps the ranks of up to 512 rows; of more rows they are found
// again.  Then tiles, and items of up to item_tiles of them.
extern "C" __global__ __launch_bounds__(1024) void nh_lora_plan_kernel(LoraPlanArgs a) {
    extern __shared__ int plan_lds[];  // [waves][G] rows of the wave, then its next slot; [G] totals, tiles and items before
    const int G = a.adapters + 1, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
    int *total = plan_lds + waves * G, *tile0 = total + G, *item0 = tile0 + G, *partial0 = item0 + G;
    for (int i = tid; i < waves * G; i += blockDim.x) plan_lds[i] = 0;
    int* mine = plan_lds + wave * G;
    const int64_t per = ((int64_t)a.m + 64 * waves - 1) / (64 * waves) * 64;
    const int r0 = (int)min((int64_t)a.m, wave * per), r1 = (int)min((int64_t)a.m, r0 + per);
    constexpr int kHeld = 8;
    const bool held = per <= 64 * kHeld;
    int bits = 0;
    while ((1 << bits) < G) ++bits;
    auto group = [&](int r) {
        if (r >= r1) return -1;
        const int e = a.ids[r];
        return e < 0 || e >= a.adapters ? a.adapters : e;
    };
    // the row's rank among the wave's rows of its adapter so far, or (counted before) its slot
    auto place = [&](int e) {
        uint64_t same = __ballot(e >= 0);
        for (int b = 0; b < bits; ++b) {
            const uint64_t bal = __ballot(e >= 0 && ((e >> b) & 1));
            same &= ((e >> b) & 1) ? bal : ~bal;
        }
        const int leader = e >= 0 ? __ffsll((unsigned long long)same) - 1 : 0;
        int at = 0;
        if (e >= 0 && lane == leader) at = atomicAdd(&mine[e], __popcll(same));
        return __shfl(at, leader, kWave) + __popcll(same & ((1ull << lane) - 1));
    };
    int e[kHeld], rank[kHeld];
    if (held) {
#pragma unroll
        for (int u = 0; u < kHeld; ++u) e[u] = group(r0 + 64 * u + lane);
    }
    __syncthreads();
    if (held) {
#pragma unroll
        for (int u = 0; u < kHeld; ++u)
            if (r0 + 64 * u < r1) rank[u] = place(e[u]);
    } else {
        for (int r = r0; r < r1; r += 64) place(group(r + lane));
    }
    __syncthreads();
    for (int i = tid; i < G; i += blockDim.x) {
        int sum = 0;
        for (int w = 0; w < waves; ++w) {
            const int n = plan_lds[w * G + i];
            plan_lds[w * G + i] = sum;
            sum += n;
        }
        total[i] = sum;
    }
    __syncthreads();
    if (wave == 0) {
        int tiles = 0, items = 0, partials = 0;
        for (int base = 0; base < G; base += 64) {
            const int i = base + lane;
            const int t = i < G ? (total[i] + kTileRows - 1) / kTileRows : 0;
            const int it = i < a.adapters ? (t + a.item_tiles - 1) / a.item_tiles : 0, pt = it > 1 ? it : 0;
            int ti = t, ii = it, pi = pt;  // inclusive scans
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const int x = __shfl_up(ti, off, kWave), y = __shfl_up(ii, off, kWave), z = __shfl_up(pi, off, kWave);
                if (lane >= off) {
                    ti += x;
                    ii += y;
                    pi += z;
                }
            }
            if (i < G) {
                tile0[i] = tiles + ti - t;
                item0[i] = items + ii - it;
                partial0[i] = partials + pi - pt;
                if (i < a.adapters && a.items) {
                    a.per_adapter[2 * i] = it;
                    a.per_adapter[2 * i + 1] = partials + pi - pt;
                }
            }
            tiles += __builtin_amdgcn_readlane(ti, 63);
            items += __builtin_amdgcn_readlane(ii, 63);
            partials += __builtin_amdgcn_readlane(pi, 63);
        }
        if (lane == 0) {
            a.counts[0] = tiles;
            a.counts[1] = items;
        }
    }
    __syncthreads();
    if (held) {
#pragma unroll
        for (int u = 0; u < kHeld; ++u) {
            const int r = r0 + 64 * u + lane;
            if (r < r1) a.slot_row[tile0[e[u]] * kTileRows + mine[e[u]] + rank[u]] = r;
        }
    } else {
        for (int r = r0; r < r1; r += 64) {  // uniform per wave
            const int g = group(r + lane), at = place(g);
            if (g >= 0) a.slot_row[tile0[g] * kTileRows + at] = r + lane;
        }
    }
    for (int i = wave; i < G; i += waves) {
        const int n = total[i], t = (n + kTileRows - 1) / kTileRows, it = (t + a.item_tiles - 1) / a.item_tiles;
        for (int j = lane; j < t; j += 64) {
            a.tile_adapter[tile0[i] + j] = i;
            if (i < a.adapters && a.items && j % a.item_tiles == 0) {
                int32_t* p = a.items + 4 * (int64_t)(item0[i] + j / a.item_tiles);
                p[0] = i;
                p[1] = tile0[i] + j;
                p[2] = min(a.item_tiles, t - j);
                p[3] = it > 1 ? partial0[i] + j / a.item_tiles : -1;
            }
        }
        if (n + lane < t * kTileRows) a.slot_row[tile0[i] * kTileRows + n + lane] = -1;
    }
}

// The low-rank values by slot, for the outer products: h as given or the sum of
// shrink's parts, times the adapter's scale; zeros where there is no row or rank.
// A tile per workgroup, 16 ranks at a time turned in LDS.
extern "C" __global__ __launch_bounds__(256) void nh_lora_finish_kernel(LoraArgs a) {
    __shared__ float turned[16][kTileRows + 1];
    const int tile = blockIdx.x;
    if (tile >= a.counts[0]) return;
    const int adapter = a.tile_adapter[tile];
    if (adapter == a.adapters) return;
    const float scale = a.scaled && a.scales ? a.scales[adapter] : 1.0f;
    const bool bf16 = a.x_dtype == DT_BF16;
    const int slot = threadIdx.x >> 2, r4 = 4 * (threadIdx.x & 3), row = a.slot_row[(int64_t)tile * kTileRows + slot];
    for (int r0 = 16 * blockIdx.y; r0 < a.rank_pad; r0 += 16 * gridDim.y) {
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (row >= 0) {
            if (a.h) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (r0 + r4 + i < a.rank) v[i] = a.h[(int64_t)row * a.rank + r0 + r4 + i];
            } else {
                const float* p = a.part + (int64_t)row * a.rank_pad + r0 + r4;
                for (int s = 0; s < a.splits; ++s) {
                    const v4f t = *(const v4f*)(p + (int64_t)s * a.m * a.rank_pad);
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = s == 0 ? t[i] : v[i] + t[i];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) turned[r4 + i][slot] = row >= 0 && r0 + r4 + i < a.rank ? v[i] * scale : 0.0f;
        __syncthreads();
        const int rank = threadIdx.x >> 4, s4 = 4 * (threadIdx.x & 15);
        const int64_t at = (r0 + rank) * a.slots + (int64_t)tile * kTileRows + s4;
        float u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = turned[rank][s4 + i];
        if (bf16) {
#pragma unroll
            for (int q = 0; q < 3; ++q) {
                const uint32_t p0 = bf16_part(u[0]), p1 = bf16_part(u[1]), p2 = bf16_part(u[2]), p3 = bf16_part(u[3]);
                *(uint2*)((uint16_t*)a.ht + (int64_t)q * a.rank_pad * a.slots + at) = make_uint2(p0 | (p1 << 16), p2 | (p3 << 16));
            }
        } else {
            *(float4*)((float*)a.ht + at) = make_float4(u[0], u[1], u[2], u[3]);
        }
        __syncthreads();
    }
}

// An adapter's partial sums in order; zeros for one without rows.
extern "C" __global__ __launch_bounds__(256) void nh_lora_reduce_kernel(LoraArgs a) {
    const int adapter = blockIdx.y, items = a.per_adapter[2 * adapter];
    if (items == 1 || (items == 0 && a.accumulate)) return;
    const int64_t size = (int64_t)a.rank * a.C, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= size) return;
    float* to = a.grad + adapter * size + i;
    float v = 0.0f;
    const float* p = a.gpart + (int64_t)a.per_adapter[2 * adapter + 1] * size + i;
    for (int s = 0; s < items; ++s) v += p[s * size];
    *to = a.accumulate ? *to + v : v;
}

// Compute kind (bf16, or f32 whatever the operands), a few rows or the plan's tiles
// forward, or the plan's backward (matrices the other way), ranks to 16, 32, 64, 128.
#define NH_LORA_RANKS(call, ...) call(__VA_ARGS__, 1) call(__VA_ARGS__, 2) call(__VA_ARGS__, 4) call(__VA_ARGS__, 8)
#define NH_CALL(kind, Frag, rows, FEW, BACK, RT)                                                                     \
    extern "C" __global__ __launch_bounds__(RT == 8 ? 256 : 512) void                                               \
    nh_lora_shrink_##kind##_##rows##_##RT##_kernel(LoraArgs a) {                                                     \
        lora_shrink<Frag, FEW, RT, BACK>(a);                                                                         \
    }                                                                                                                \
    extern "C" __global__ __launch_bounds__(256) void nh_lora_expand_##kind##_##rows##_##RT##_kernel(LoraArgs a) {    \
        lora_expand<Frag, FEW, RT, !BACK>(a);                                                                        \
    }
NH_LORA_RANKS(NH_CALL, bf16, Frag16, few, true, false)
NH_LORA_RANKS(NH_CALL, bf16, Frag16, tiles, false, false)
NH_LORA_RANKS(NH_CALL, bf16, Frag16, back, false, true)
NH_LORA_RANKS(NH_CALL, f32, Frag32, few, true, false)
NH_LORA_RANKS(NH_CALL, f32, Frag32, tiles, false, false)
NH_LORA_RANKS(NH_CALL, f32, Frag32, back, false, true)
#undef NH_CALL
#define NH_CALL(kind, Frag, name, COLS, RT)                                                                           \
    extern "C" __global__ __launch_bounds__(256) void nh_lora_outer_##kind##_##name##_##RT##_kernel(LoraArgs a) {      \
        lora_outer<Frag, RT, COLS>(a);                                                                               \
    }
NH_LORA_RANKS(NH_CALL, bf16, Frag16, a, false)
NH_LORA_RANKS(NH_CALL, bf16, Frag16, b, true)
NH_LORA_RANKS(NH_CALL, f32, Frag32, a, false)
NH_LORA_RANKS(NH_CALL, f32, Frag32, b, true)
#undef NH_CALL
#undef NH_LORA_RANKS
