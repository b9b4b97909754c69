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
    v4i v;
};
struct Frag32 {
    float v[8];
};

// Eight consecutive values, `n` of them there (zeros behind).
__device__ __forceinline__ void load8(const uint16_t* p, int n, Frag16& f) {
    if (n >= 8) {
        __builtin_memcpy(&f.v, p, 16);
    } else {
        uint32_t u[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = i < n ? p[i] : 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i) f.v[i] = (int)(u[2 * i] | (u[2 * i + 1] << 16));
    }
}

__device__ __forceinline__ void load8(const void* p, int64_t at, int dtype, int n, Frag16& f) {
    load8((const uint16_t*)p + at, n, f);
}

__device__ __forceinline__ void load8(const void* p, int64_t at, int dtype, int n, Frag32& f) {
    if (dtype == DT_BF16) {
        Frag16 h;
        load8((const uint16_t*)p + at, n, h);
        unpack_bf16x8(h.v, f.v);
    } else {
        const float* q = (const float*)p + at;
        if (n >= 8) {
            __builtin_memcpy(f.v, q, 32);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) f.v[i] = i < n ? q[i] : 0.0f;
        }
    }
}

// Eight values `stride` apart, the i-th there if ok(i).
template <class Ok>
__device__ __forceinline__ void load8s(const void* p, int64_t at, int64_t stride, int dtype, Ok ok, Frag16& f) {
    const uint16_t* q = (const uint16_t*)p + at;
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = ok(i) ? q[i * stride] : 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) f.v[i] = (int)(u[2 * i] | (u[2 * i + 1] << 16));
}

template <class Ok>
__device__ __forceinline__ void load8s(const void* p, int64_t at, int64_t stride, int dtype, Ok ok, Frag32& f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f.v[i] = ok(i) ? load_as_f32(p, at + i * stride, dtype) : 0.0f;
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
// many (0: nothing to do), uniform.  64 at a time from the plan, or 16 of at most
// 64 rows in all, where every row that is the 1st, 17th, .. of its adapter leads a
// tile (RB = 1).
template <int RB>
__device__ __forceinline__ int lora_tile(const LoraArgs& a, int tile, int* rows, int& adapter) {
    const int lane = threadIdx.x & 63;
    if constexpr (RB == 1) {
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
        static_assert(16 * RB == kTileRows, "a tile of the plan");
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
// Waves of a workgroup take consecutive parts of the columns and add up through
// LDS; ranks past the last and rows past the tile's are computed on the nearest
// valid operand and not read again, columns past C are zeros in both operands.
template <class Frag, int RB, int RT>
__device__ __forceinline__ void lora_shrink(const LoraArgs& a) {
    extern __shared__ float lora_lds[];  // [waves][16 RB][16 RT]
    __shared__ int rows[16 * RB];
    int adapter;
    const int count = lora_tile<RB>(a, blockIdx.x, rows, adapter);
    if (count == 0 || adapter == a.adapters) return;  // uniform
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, g = lane >> 4, l16 = lane & 15;
    const int64_t first = ((int64_t)blockIdx.y * waves + wave) * a.per_wave;
    const int c0 = (int)min((int64_t)a.C, first), c1 = min(a.C, c0 + a.per_wave);
    int64_t xat[RB], wat[RT];
#pragma unroll
    for (int b = 0; b < RB; ++b) xat[b] = (int64_t)rows[min(16 * b + l16, count - 1)] * a.C;
    const int64_t matrix = (int64_t)adapter * a.rank * a.C;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int rank = min(16 * r + l16, a.rank - 1);
        wat[r] = matrix + (a.w_cols ? rank : (int64_t)rank * a.C);
    }
    v4f acc[RB][RT];
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int r = 0; r < RT; ++r) acc[b][r] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    for (int c = c0; c < c1; c += 32) {
        const int at = c + 8 * g, n = a.C - at;  // n may be past the end: zeros
        Frag x[RB], w[RT];
#pragma unroll
        for (int b = 0; b < RB; ++b)
            if (16 * b < count) load8(a.x, xat[b] + at, a.x_dtype, n, x[b]);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            if (a.w_cols)
                load8s(a.w, wat[r] + (int64_t)at * a.rank, a.rank, a.w_dtype, [&](int i) { return i < n; }, w[r]);
            else
                load8(a.w, wat[r] + at, a.w_dtype, n, w[r]);
        }
#pragma unroll
        for (int b = 0; b < RB; ++b)
            if (16 * b < count) {
#pragma unroll
                for (int r = 0; r < RT; ++r) acc[b][r] = mma(w[r], x[b], acc[b][r]);
            }
    }
    constexpr int kPlane = 256 * RB * RT;
    float* mine = lora_lds + wave * kPlane;
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int r = 0; r < RT; ++r) *(v4f*)(mine + (16 * b + l16) * 16 * RT + 16 * r + 4 * g) = acc[b][r];
    __syncthreads();
    for (int i = 4 * threadIdx.x; i < count * 16 * RT; i += 4 * blockDim.x) {
        v4f v = *(v4f*)(lora_lds + i);
        for (int w = 1; w < waves; ++w) v += *(v4f*)(lora_lds + w * kPlane + i);
        const int row = rows[i / (16 * RT)];
        *(v4f*)(a.part + ((int64_t)blockIdx.y * a.m + row) * (16 * RT) + i % (16 * RT)) = v;
    }
}

// ---- expand --------------------------------------------------------------------
// out[row][c] = base[row][c] + sum over ranks of (s) h[row][rank] w(rank, c), h the
// sum of shrink's parts in order.  Per wave and turn 32 columns as two tiles whose
// columns interleave by fours, so that a lane's results are eight consecutive ones.
template <class Frag, class Split, int RB, int RT>
__device__ __forceinline__ void lora_expand_columns(const LoraArgs& a, const int* rows, const float* hs, int count,
                                                    int adapter, int c0, int c1) {
    constexpr int KC = (RT + 1) / 2;  // steps of 32 ranks
    const int lane = threadIdx.x & 63, g = lane >> 4, l16 = lane & 15;
    Split h[RB][KC];
    int64_t at[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const int row = min(16 * b + l16, count - 1);
        at[b] = (int64_t)rows[row] * a.C;
#pragma unroll
        for (int q = 0; q < KC; ++q) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 32 * q + 8 * g < 16 * RT ? hs[row * 16 * RT + 32 * q + 8 * g + i] : 0.0f;
            split8(v, h[b][q]);
        }
    }
    const int64_t matrix = (int64_t)adapter * a.rank * a.C;
    for (int c = c0; c < c1; c += 32) {
        Frag w[2][KC];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const int col = min(c + 8 * (l16 >> 2) + 4 * p + (l16 & 3), a.C - 1);
#pragma unroll
            for (int q = 0; q < KC; ++q) {
                const int rank = 32 * q + 8 * g, n = a.rank - rank;
                if (a.w_cols)
                    load8(a.w, matrix + (int64_t)col * a.rank + rank, a.w_dtype, n, w[p][q]);
                else
                    load8s(a.w, matrix + (int64_t)rank * a.C + col, a.C, a.w_dtype, [&](int i) { return i < n; }, w[p][q]);
            }
        }
        const int first = c + 8 * g, there = a.C - first;
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            if (16 * b >= count) continue;  // uniform
            v4f acc[2];
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                acc[p] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int s = Split::parts - 1; s >= 0; --s)  // the small parts first
#pragma unroll
                    for (int q = 0; q < KC; ++q) acc[p] = mma(w[p][q], h[b][q].f[s], acc[p]);
            }
            if (16 * b + l16 >= count || there <= 0) continue;
            float v[8];
            Frag32 base;
            if (a.base) {
                load8(a.base, at[b] + first, a.out_dtype, there, base);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) base.v[i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = base.v[i] + acc[i >> 2][i & 3];
            if (there >= 8) {
                if (a.out_dtype == DT_BF16) {
                    const uint32_t u[4] = {f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3]),
                                           f32x2_to_bf16x2(v[4], v[5]), f32x2_to_bf16x2(v[6], v[7])};
                    __builtin_memcpy((uint16_t*)a.out + at[b] + first, u, 16);
                } else {
                    __builtin_memcpy((float*)a.out + at[b] + first, v, 32);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < there) store_out(a.out, at[b] + first + i, v[i], a.out_dtype);
            }
        }
    }
}

template <class Frag, int RB, int RT>
__device__ __forceinline__ void lora_expand(const LoraArgs& a) {
    __shared__ int rows[16 * RB];
    __shared__ float hs[256 * RB * RT];
    int adapter;
    const int count = lora_tile<RB>(a, blockIdx.x, rows, adapter);
    if (count == 0) return;  // uniform
    const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int64_t wide = (int64_t)waves * a.per_wave, start = min((int64_t)a.C, blockIdx.y * wide);
    if (adapter == a.adapters) {  // rows without an adapter: the base
        const int end = (int)min((int64_t)a.C, start + wide);
        if (blockIdx.y == 0 && a.h_out)
            for (int i = threadIdx.x; i < count * a.rank; i += blockDim.x)
                a.h_out[(int64_t)rows[i / a.rank] * a.rank + i % a.rank] = 0.0f;
        if (a.base == a.out) return;
        for (int r = 0; r < count; ++r) {
            const int64_t at = (int64_t)rows[r] * a.C;
            for (int c = (int)start + threadIdx.x; c < end; c += blockDim.x)
                store_out(a.out, at + c, a.base ? load_as_f32(a.base, at + c, a.out_dtype) : 0.0f, a.out_dtype);
        }
        return;
    }
    const float scale = a.scaled && a.scales ? a.scales[adapter] : 1.0f;
    for (int i = threadIdx.x; i < count * 16 * RT; i += blockDim.x) {
        const int row = rows[i / (16 * RT)], rank = i % (16 * RT);
        float v = 0.0f;
        if (rank < a.rank) {
            const float* p = a.part + (int64_t)row * (16 * RT) + rank;
            v = p[0];
            for (int s = 1; s < a.splits; ++s) v += p[(int64_t)s * a.m * (16 * RT)];
            if (blockIdx.y == 0 && a.h_out) a.h_out[(int64_t)row * a.rank + rank] = v;
            v *= scale;
        }
        hs[i] = v;
    }
    __syncthreads();
    const int c0 = (int)min((int64_t)a.C, start + (int64_t)wave * a.per_wave), c1 = min(a.C, c0 + a.per_wave);
    if constexpr (sizeof(Frag) == sizeof(Frag32)) {
        lora_expand_columns<Frag, Split32, RB, RT>(a, rows, hs, count, adapter, c0, c1);
    } else if (a.out_dtype == DT_BF16) {
        lora_expand_columns<Frag, Split16<2>, RB, RT>(a, rows, hs, count, adapter, c0, c1);
    } else {
        lora_expand_columns<Frag, Split16<3>, RB, RT>(a, rows, hs, count, adapter, c0, c1);
    }
}

// ---- outer ---------------------------------------------------------------------
// grad(rank, c) of an adapter = sum over its rows of ht[rank][slot] x[row][c].  An
// item of the plan is some of an adapter's tiles; one that has them all writes the
// gradient, the others a partial sum each.  64 columns per wave.
template <class Frag, int RT>
__device__ __forceinline__ void lora_outer(const LoraArgs& a) {
    constexpr bool kBf16 = sizeof(Frag) == sizeof(Frag16);
    constexpr int PARTS = kBf16 ? 3 : 1, CT = 4;
    if ((int)blockIdx.y >= a.counts[1]) return;
    const int32_t* item = a.items + 4 * blockIdx.y;
    const int adapter = item[0], tile = item[1], tiles = item[2], partial = item[3];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, l16 = lane & 15;
    const int64_t first = ((int64_t)blockIdx.x * (blockDim.x >> 6) + wave) * 16 * CT;
    if (first >= a.C) return;
    const int c0 = (int)first;
    v4f acc[CT][RT];
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int r = 0; r < RT; ++r) acc[c][r] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    const int64_t s0 = (int64_t)tile * kTileRows, s1 = s0 + (int64_t)tiles * kTileRows;
    for (int64_t s = s0; s < s1; s += 32) {
        const int64_t at = s + 8 * g;
        int row[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) row[i] = a.slot_row[at + i];
        Frag x[CT], h[RT][PARTS];
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            const int col = min(c0 + 16 * c + l16, a.C - 1);
            if constexpr (kBf16) {
                uint32_t u[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) u[i] = row[i] >= 0 ? ((const uint16_t*)a.x)[(int64_t)row[i] * a.C + col] : 0u;
#pragma unroll
                for (int i = 0; i < 4; ++i) x[c].v[i] = (int)(u[2 * i] | (u[2 * i + 1] << 16));
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    x[c].v[i] = row[i] >= 0 ? load_as_f32(a.x, (int64_t)row[i] * a.C + col, a.x_dtype) : 0.0f;
            }
        }
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
                load8(a.ht, ((int64_t)p * (16 * RT) + 16 * r + l16) * a.slots + at, DT_F32, 8, h[r][p]);
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int p = PARTS - 1; p >= 0; --p)
                    acc[c][r] = a.w_cols ? mma(h[r][p], x[c], acc[c][r]) : mma(x[c], h[r][p], acc[c][r]);
    }
    const bool add = partial < 0 && a.accumulate;
    float* to = partial < 0 ? a.grad + (int64_t)adapter * a.rank * a.C : a.gpart + (int64_t)partial * a.rank * a.C;
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            // w_cols: the lane's column, four ranks; else the lane's rank, four columns
            const int col = c0 + 16 * c + (a.w_cols ? l16 : 4 * g), rank = 16 * r + (a.w_cols ? 4 * g : l16);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int cc = a.w_cols ? col : col + i, rr = a.w_cols ? rank + i : rank;
                if (cc >= a.C || rr >= a.rank) continue;
                float* p = to + (a.w_cols ? (int64_t)cc * a.rank + rr : (int64_t)rr * a.C + cc);
                *p = add ? *p + acc[c][r][i] : acc[c][r][i];
            }
        }
}

}  // namespace

// ---- the plan ------------------------------------------------------------------
// One workgroup sorts the rows by adapter, stable by row, rows without one last,
// each adapter's from a tile of its own on; the waves take consecutive parts of
// the rows.  Then tiles, and items of up to item_tiles of them.
extern "C" __global__ __launch_bounds__(1024) void nh_lora_plan_kernel(LoraPlanArgs a) {
    extern __shared__ int plan_lds[];  // [waves][G] rows of the wave, then its next slot; [G] totals
    const int G = a.adapters + 1, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
    int* total = plan_lds + waves * G;
    for (int i = tid; i < waves * G; i += blockDim.x) plan_lds[i] = 0;
    __syncthreads();
    int* mine = plan_lds + wave * G;
    const int64_t per = ((int64_t)a.m + 64 * waves - 1) / (64 * waves) * 64;
    const int r0 = (int)min((int64_t)a.m, wave * per), r1 = (int)min((int64_t)a.m, r0 + per);
    auto group = [&](int r) {
        if (r >= r1) return -1;
        const int e = a.ids[r];
        return e < 0 || e >= a.adapters ? a.adapters : e;
    };
    for (int r = r0 + lane; r < r1; r += 64) atomicAdd(&mine[group(r)], 1);
    __syncthreads();
    for (int e = tid; e < G; e += blockDim.x) {
        int sum = 0;
        for (int w = 0; w < waves; ++w) sum += plan_lds[w * G + e];
        total[e] = sum;
    }
    __syncthreads();
    if (wave == 0) {
        int tiles = 0, items = 0, partials = 0;
        for (int base = 0; base < G; base += 64) {
            const int e = base + lane;
            const int n = e < G ? total[e] : 0, t = (n + kTileRows - 1) / kTileRows;
            const int it = e < a.adapters ? (t + a.item_tiles - 1) / a.item_tiles : 0, pt = it > 1 ? it : 0;
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
            const int tile = tiles + ti - t, item = items + ii - it, partial = partials + pi - pt;
            if (e < G) {
                for (int i = 0; i < t; ++i) a.tile_adapter[tile + i] = e;
                for (int i = n; i < t * kTileRows; ++i) a.slot_row[(int64_t)tile * kTileRows + i] = -1;
                if (e < a.adapters && a.items) {
                    for (int i = 0; i < it; ++i) {
                        int32_t* p = a.items + 4 * (int64_t)(item + i);
                        p[0] = e;
                        p[1] = tile + i * a.item_tiles;
                        p[2] = min(a.item_tiles, t - i * a.item_tiles);
                        p[3] = it > 1 ? partial + i : -1;
                    }
                    a.per_adapter[2 * e] = it;
                    a.per_adapter[2 * e + 1] = partial;
                }
                int slot = tile * kTileRows;
                for (int w = 0; w < waves; ++w) {
                    const int c = plan_lds[w * G + e];
                    plan_lds[w * G + e] = slot;
                    slot += c;
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
    int bits = 0;
    while ((1 << bits) < G) ++bits;
    for (int base = r0; base < r1; base += 64) {  // uniform per wave
        const int r = base + lane, e = group(r);
        uint64_t same = __ballot(e >= 0);
        for (int b = 0; b < bits; ++b) {
            const uint64_t bal = __ballot(e >= 0 && ((e >> b) & 1));
            same &= ((e >> b) & 1) ? bal : ~bal;
        }
        const int leader = e >= 0 ? __ffsll((unsigned long long)same) - 1 : 0;
        int slot = 0;
        if (e >= 0 && lane == leader) slot = atomicAdd(&mine[e], __popcll(same));
        slot = __shfl(slot, leader, kWave);
        if (e >= 0) a.slot_row[slot + __popcll(same & ((1ull << lane) - 1))] = r;
    }
}

// The low-rank values by slot, for the outer products: h as given or the sum of
// shrink's parts, times the adapter's scale; zeros where there is no row or rank.
extern "C" __global__ __launch_bounds__(256) void nh_lora_finish_kernel(LoraArgs a) {
    const int tile = blockIdx.x;
    if (tile >= a.counts[0]) return;
    const int adapter = a.tile_adapter[tile];
    if (adapter == a.adapters) return;
    const float scale = a.scaled && a.scales ? a.scales[adapter] : 1.0f;
    const bool bf16 = a.x_dtype == DT_BF16;
    for (int i = threadIdx.x; i < kTileRows * a.rank_pad; i += blockDim.x) {
        const int64_t slot = (int64_t)tile * kTileRows + (i & (kTileRows - 1));
        const int rank = i / kTileRows, row = a.slot_row[slot];
        float v = 0.0f;
        if (row >= 0 && rank < a.rank) {
            if (a.h) {
                v = a.h[(int64_t)row * a.rank + rank];
            } else {
                const float* p = a.part + (int64_t)row * a.rank_pad + rank;
                v = p[0];
                for (int s = 1; s < a.splits; ++s) v += p[(int64_t)s * a.m * a.rank_pad];
            }
            v *= scale;
        }
        const int64_t at = rank * a.slots + slot;
        if (bf16) {
#pragma unroll
            for (int q = 0; q < 3; ++q) ((uint16_t*)a.ht)[(int64_t)q * a.rank_pad * a.slots + at] = (uint16_t)bf16_part(v);
        } else {
            ((float*)a.ht)[at] = v;
        }
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

// Compute kind (bf16, or f32 whatever the operands), 16 rows or 64, ranks to 16, 32, 64, 128.
#define NH_LORA_FORMS(call) \
    call(bf16, Frag16, 1, 1) call(bf16, Frag16, 1, 2) call(bf16, Frag16, 1, 4) call(bf16, Frag16, 1, 8) \
    call(bf16, Frag16, 4, 1) call(bf16, Frag16, 4, 2) call(bf16, Frag16, 4, 4) call(bf16, Frag16, 4, 8) \
    call(f32, Frag32, 1, 1) call(f32, Frag32, 1, 2) call(f32, Frag32, 1, 4) call(f32, Frag32, 1, 8) \
    call(f32, Frag32, 4, 1) call(f32, Frag32, 4, 2) call(f32, Frag32, 4, 4) call(f32, Frag32, 4, 8)
#define NH_CALL(kind, Frag, RB, RT)                                                                                  \
    extern "C" __global__ __launch_bounds__(256) void nh_lora_shrink_##kind##_##RB##_##RT##_kernel(LoraArgs a) {      \
        lora_shrink<Frag, RB, RT>(a);                                                                                \
    }                                                                                                                \
    extern "C" __global__ __launch_bounds__(256) void nh_lora_expand_##kind##_##RB##_##RT##_kernel(LoraArgs a) {      \
        lora_expand<Frag, RB, RT>(a);                                                                                \
    }
NH_LORA_FORMS(NH_CALL)
#undef NH_CALL
#define NH_CALL(kind, Frag, RT)                                                                                       \
    extern "C" __global__ __launch_bounds__(256) void nh_lora_outer_##kind##_##RT##_kernel(LoraArgs a) {               \
        lora_outer<Frag, RT>(a);                                                                                     \
    }
NH_CALL(bf16, Frag16, 1) NH_CALL(bf16, Frag16, 2) NH_CALL(bf16, Frag16, 4) NH_CALL(bf16, Frag16, 8)
NH_CALL(f32, Frag32, 1) NH_CALL(f32, Frag32, 2) NH_CALL(f32, Frag32, 4) NH_CALL(f32, Frag32, 8)
#undef NH_CALL
#undef NH_LORA_FORMS
