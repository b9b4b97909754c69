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
// sums.  All three go in, whatever the result's type: where terms or the base cancel,
// what two parts leave out (2^-15 of a term) is more than a bf16 result's own
// rounding.  Otherwise the f32 matrix cores take every value as it is.  Every sum
// has a fixed order: results do not change from run to run.
//
// A row's products see its own values only; what stands in rows without an
// adapter, or in another adapter's matrices, reaches no other row.
#include "nh_device.h"

using namespace nh;

namespace {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4), aligned(2)));

constexpr int kTileRows = 64;  // slots per tile of the plan

// A choice made where a body is built.
template <bool B>
struct Choice {
    static constexpr bool value = B;
};
typedef Choice<true> Yes;
typedef Choice<false> No;

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

// acc of products with the parts of h after the first, which are zero where few bits or
// no finite value are left: beside an infinity they say NaN.  An operand that is not
// finite makes the first part's product infinite or NaN as the formula has it (only
// values under 2^-133 have no first part), so what comes ahead of it is held finite
// (med3 of a NaN is the least of the others).
__device__ __forceinline__ v4f held_finite(v4f acc) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = __builtin_amdgcn_fmed3f(acc[i], -3.402823466e38f, 3.402823466e38f);
    return acc;
}

// The same where the sum goes on: operands for those parts, with zeros for what is not finite.
__device__ __forceinline__ Frag16 finite_values(const Frag16& f) {
    Frag16 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t u = (uint32_t)f.v[i], e = u & 0x7f807f80u;
        const uint32_t lo = (e & 0xffffu) == 0x7f80u ? 0u : u, hi = e >> 16 == 0x7f80u ? 0u : u;
        r.v[i] = (int)((lo & 0xffffu) | (hi & 0xffff0000u));
    }
    return r;
}
__device__ __forceinline__ const Frag32& finite_values(const Frag32& f) { return f; }

// The sum of w h over K, of h's parts the small ones first.
template <class Frag, int KC, int PARTS>
__device__ __forceinline__ v4f mma_parts(const Frag (&w)[KC], const Frag (&h)[KC][PARTS]) {
    v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = PARTS - 1; s >= 0; --s) {
#pragma unroll
        for (int q = 0; q < KC; ++q) acc = mma(w[q], h[q][s], acc);
        if (s == 1) acc = held_finite(acc);
    }
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

// The three bf16 parts of two values, a pair a part.  A value that is not finite is its
// first part, with zeros behind (canonical: a NaN's upper half is one as well).
__device__ __forceinline__ void bf16_parts(float a, float b, uint32_t (&parts)[3]) {
    auto pair = [](float lo, float hi) { return f32_bits(lo) >> 16 | (f32_bits(hi) & 0xffff0000u); };
    auto rest = [](float v) { return v - f32_from_bits(f32_bits(v) & 0xffff0000u); };  // exact
    a = __builtin_canonicalizef(a);
    b = __builtin_canonicalizef(b);
    parts[0] = pair(a, b);
    a = __builtin_isfinite(a) ? rest(a) : 0.0f;
    b = __builtin_isfinite(b) ? rest(b) : 0.0f;
    parts[1] = pair(a, b);
    parts[2] = pair(rest(a), rest(b));
}

// ---- the rows of a workgroup ---------------------------------------------------
// Of at most 64 rows in all every one that is the 1st, 17th, .. of its adapter leads
// 16: the adapter (`adapters`: none) and the rows of the 16 that a workgroup is for,
// returning how many (0: none), uniform.  With a workgroup for each row (many
// adapters) that is the row to lead; with fewer the number of the leader, which costs
// a ballot per bit of the adapters first (0.25 us of a launch).
__device__ __forceinline__ int lora_few(const LoraArgs& a, int number, int* rows, int& adapter) {
    const int lane = threadIdx.x & 63;
    int e = -1;
    if (lane < a.m) {
        e = a.ids[lane];
        if (e < 0 || e >= a.adapters) e = a.adapters;
    }
    const uint64_t lower = (1ull << lane) - 1;
    int lead = number;
    if (a.numbered) {
        uint64_t same = __ballot(e >= 0);  // the lanes of the same adapter
        for (int bit = 1; bit <= a.adapters; bit <<= 1) {
            const uint64_t with = __ballot(e & bit);
            same &= (e & bit) ? with : ~with;
        }
        const uint64_t leads = __ballot(e >= 0 && __popcll(same & lower) % 16 == 0);
        if (number >= __popcll(leads)) return 0;  // uniform
        lead = __ffsll((unsigned long long)__ballot(((leads >> lane) & 1) && __popcll(leads & lower) == number)) - 1;
    }
    adapter = __builtin_amdgcn_readlane(e, lead);
    const uint64_t group = __ballot(e == adapter);
    const int before = __popcll(group & ((1ull << lead) - 1)), mine = __popcll(group & lower) - before;
    if (before % 16 != 0) return 0;  // uniform
    if (threadIdx.x < 64 && e == adapter && mine >= 0 && mine < 16) rows[mine] = lane;
    __syncthreads();
    return min(16, __popcll(group) - before);
}

// Consecutive shares of n, to the workgroups of an XCD one after the other
// (workgroups go round the eight of them, the grid being a multiple): what shares an
// adapter's matrix reads it into one L2.
__device__ __forceinline__ int xcd_order(int block, int blocks) { return (block & 7) * (blocks >> 3) + (block >> 3); }

// ---- shrink --------------------------------------------------------------------
// part[split][row][rank] = sum over the split's columns of x[row][c] w(rank, c), for
// 16 rows of an adapter.  The waves take consecutive parts of the columns and add up
// through LDS; there is one split unless rows are few, so that rows are read once,
// and the matrix, which all of an adapter's rows share, from the L2s.
// Ranks past the last and rows past the tile's are computed on the nearest valid
// operand and not read again; columns past C are zeros in both operands.
// bf16 goes through LDS, a wave's part of it: the operands' layout has neighbouring
// lanes in different rows, and a load costs the address unit a turn for each piece
// that neighbouring lanes do not continue (8192 x 4096, rank 32: 37 us straight into
// registers).  So a load has 8 rows of 64 columns, 8 lanes a row, and LDS turns it.
// A matrix of [C][rank] (COLS) is read as it lies and turned by transposing reads,
// for ranks that are multiples of 8.
// 4096 rows of 4096, rank 64: 25 us, of which a launch without loads or turning takes
// 10, one without the matrix's loads 18, one without the rows' 18.5; 8192 rows, rank
// 32: 28 us (67 MB of rows, 134 MB of matrix from the L2s).  What bounds it is a
// workgroup's chain (plan, rows, four blocks, the sum over waves), one round of them.
template <class Frag, bool FEW, int RT, bool COLS>
struct ShrinkForm {
    static constexpr bool staged = Frag::bf16;
    static constexpr int RP = 16 * RT;
    // columns in flight: loads of 10 to 18 KiB a wave
    static constexpr int block = !Frag::bf16 ? 32 : RT <= 2 ? 128 : 64;
    static constexpr int pitch = 64 + 8;  // of 16 rows of 64 columns: sixteen rows' reads meet no bank twice
    // a wave's LDS: 16 rows, and two times 16 more or 32 rows of [C][rank]
    static constexpr int values = !staged ? 0 : COLS ? 16 * pitch + 64 * RP : 3 * 16 * pitch;
};

template <class Frag, bool FEW, int RT, bool COLS>
__device__ __forceinline__ void lora_shrink(const LoraArgs& a) {
    using F = ShrinkForm<Frag, FEW, RT, COLS>;
    constexpr int RP = F::RP, kPlane = 16 * RP;
    extern __shared__ float lora_lds[];  // half the waves' sums; before: each wave's own part
    __shared__ int rows[16];
    int adapter, count;
    unsigned unit = blockIdx.x;
    if constexpr (FEW) {
        count = lora_few(a, blockIdx.x, rows, adapter);
        if (count == 0) return;  // uniform
    } else {
        const int tiles = a.counts[0], each = (4 * tiles + 7) / 8, order = blockIdx.x >> 3;
        unit = (blockIdx.x & 7) * each + order;  // a quarter of a tile
        if (order >= each || unit >= 4u * tiles) return;
        const int lane = threadIdx.x & 63;
        adapter = a.tile_adapter[unit >> 2];
        const int row = lane < 16 ? a.slot_row[(int64_t)unit * 16 + lane] : -1;  // those without a row are the last
        if (threadIdx.x < 16) rows[lane] = row;
        __syncthreads();
        count = __popcll(__ballot(row >= 0));
    }
    if (count == 0 || adapter == a.adapters) return;  // uniform
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = blockDim.x >> 7, g = lane >> 4, l16 = lane & 15;
    const int64_t first = ((int64_t)blockIdx.y * (blockDim.x >> 6) + wave) * a.per_wave;
    const int c0 = (int)min((int64_t)a.C, first), c1 = min(a.C, c0 + a.per_wave);
    const int64_t matrix = (int64_t)adapter * a.rank * a.C, xat = (int64_t)rows[min(l16, count - 1)] * a.C;
    int64_t wat[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int rank = min(16 * r + l16, a.rank - 1);
        wat[r] = matrix + (COLS ? rank : (int64_t)rank * a.C);
    }
    v4f acc[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) acc[r] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    uint16_t* lds = (uint16_t*)lora_lds + wave * F::values;
    // The operands of 32 columns from c on, of which the last may be past the end.
    auto load_x = [&](int c, Frag& x) {
        const int at = c + 8 * g;
        if (at + 8 <= a.C) load8(a.x, xat + at, a.x_dtype, x);
        else load8(a.x, xat + at, 1, a.x_dtype, a.C - at, x);
    };
    auto load_w = [&](int c, Frag& w, int r) {
        const int at = c + 8 * g;
        if constexpr (COLS) load8(a.w, wat[r] + (int64_t)at * a.rank, a.rank, a.w_dtype, a.C - at, w);
        else if (at + 8 <= a.C) load8(a.w, wat[r] + at, a.w_dtype, w);
        else load8(a.w, wat[r] + at, 1, a.w_dtype, a.C - at, w);
    };
    // Rows of a power of two bytes have a column all in one channel of the caches and
    // the memory, so workgroups start 128 columns apart and go round their own part.
    const int blocks = Frag::bf16 && COLS && a.rank % 8 != 0 ? 0 : (c1 - c0) / F::block;
    int at = blocks > 0 ? (int)(unit * (128u / F::block) % (unsigned)blocks) : 0;
    if constexpr (F::staged) {
        constexpr int J = F::block / 64;
        // of the u-th of a block's loads the lane's row is 8 u + lane / 8
        const int l8 = 8 * (lane & 7);
        int64_t from[2], wfrom[RT][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            from[u] = (int64_t)rows[min(8 * u + (lane >> 3), count - 1)] * a.C + l8;
#pragma unroll
            for (int r = 0; r < RT; ++r) wfrom[r][u] = matrix + (int64_t)min(16 * r + 8 * u + (lane >> 3), a.rank - 1) * a.C + l8;
        }
        uint16_t* put = lds + (lane >> 3) * F::pitch + l8;
        const uint16_t* get = lds + l16 * F::pitch + 8 * g;
        uint16_t* more = lds + 16 * F::pitch;
        auto turn = [&](const v4i (&v)[2], int region, Frag16 (&f)[2]) {  // 16 rows of 64 columns, as two operands
#pragma unroll
            for (int u = 0; u < 2; ++u) *(v4i*)(put + region * 16 * F::pitch + 8 * u * F::pitch) = v[u];
            asm volatile("" ::: "memory");  // a wave's LDS accesses go in order
#pragma unroll
            for (int u = 0; u < 2; ++u) f[u].v = *(const v4i*)(get + region * 16 * F::pitch + 32 * u);
            asm volatile("" ::: "memory");
        };
        // [C][rank]: 64 rows are 8 rank eights in a row, which go to rows of RP, the rest of
        // them zeros; the eight of load q, and where (its row by a multiplication: of fewer than
        // 1024 by at most 16 it is exact)
        const int eights = a.rank / 8, most = 8 * a.rank - 1;
        const uint32_t inverse = COLS && eights > 0 ? 65536u / eights + 1 : 0;
        auto eight = [&](int q) { return min(64 * q + lane, most); };
        auto eight_at = [&](int q) {
            const int row = (int)((uint32_t)eight(q) * inverse >> 16);
            return row * RP + 8 * (eight(q) - row * eights);
        };
        if (COLS && a.rank < RP) {
#pragma unroll
            for (int q = 0; q < 2 * RT; ++q) *(v4i*)(more + 512 * q + 8 * lane) = v4i{0, 0, 0, 0};
            asm volatile("" ::: "memory");
        }
        v4i next[J][2];  // the next block's rows, which come from memory
        auto load_rows_at = [&](int c) {
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int u = 0; u < 2; ++u) __builtin_memcpy(&next[j][u], (const uint16_t*)a.x + from[u] + c + 64 * j, 16);
        };
        if (blocks > 0) load_rows_at(c0 + F::block * at);
        for (int n = 0; n < blocks; ++n) {
            const int c = c0 + F::block * at;
            if (++at == blocks) at = 0;
            v4i x[J][2], w[J][RT][2];
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    x[j][u] = next[j][u];
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        const int64_t p = COLS ? matrix + (int64_t)(c + 64 * j) * a.rank + 8 * eight(2 * r + u) : wfrom[r][u] + c + 64 * j;
                        __builtin_memcpy(&w[j][r][u], (const uint16_t*)a.w + p, 16);
                    }
                }
            if constexpr (!FEW) load_rows_at(c0 + F::block * at);  // the last block's: the first again
            __builtin_amdgcn_sched_barrier(0);  // every load of the block ahead of its first wait
            if constexpr (FEW) if (n + 1 < blocks) load_rows_at(c0 + F::block * at);
#pragma unroll
            for (int j = 0; j < J; ++j) {
                Frag16 fx[2];
                turn(x[j], 0, fx);
                if constexpr (COLS) {
#pragma unroll
                    for (int r = 0; r < RT; ++r)
#pragma unroll
                        for (int u = 0; u < 2; ++u) *(v4i*)(more + eight_at(2 * r + u)) = w[j][r][u];
                    asm volatile("" ::: "memory");
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int r = 0; r < RT; ++r) {
                            Frag16 fw;
                            load_rows(more + 32 * u * RP, RP, [&](int i) { return 16 * r + i; }, fw);
                            acc[r] = mma(fw, fx[u], acc[r]);
                        }
                    asm volatile("" ::: "memory");
                } else {
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        Frag16 fw[2];
                        turn(w[j][r], 1 + (r & 1), fw);
#pragma unroll
                        for (int u = 0; u < 2; ++u) acc[r] = mma(fw[u], fx[u], acc[r]);
                    }
                }
            }
        }
    } else {
        for (int n = 0; n < blocks; ++n) {
            const int c = c0 + F::block * at;
            if (++at == blocks) at = 0;
            Frag x;
            load8(a.x, xat + c + 8 * g, a.x_dtype, x);
            constexpr int kTogether = COLS ? 2 : 4;  // rank tiles whose loads go out at once
#pragma unroll
            for (int r0 = 0; r0 < RT; r0 += kTogether) {
                Frag w[kTogether];
#pragma unroll
                for (int r = 0; r < kTogether; ++r)
                    if (r0 + r < RT) {
                        if constexpr (COLS) load8(a.w, wat[r0 + r] + (int64_t)(c + 8 * g) * a.rank, a.rank, a.w_dtype, 8, w[r]);
                        else load8(a.w, wat[r0 + r] + c + 8 * g, a.w_dtype, w[r]);
                    }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int r = 0; r < kTogether; ++r)
                    if (r0 + r < RT) acc[r0 + r] = mma(w[r], x, acc[r0 + r]);
            }
        }
    }
    for (int c = c0 + F::block * blocks; c < c1; c += 32) {
        Frag x;
        load_x(c, x);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            Frag w;
            load_w(c, w, r);
            acc[r] = mma(w, x, acc[r]);
        }
    }
    // the waves' sums: the second half's, the first half's onto them, then all in order
    if (F::staged) __syncthreads();
    float* mine = lora_lds + (wave % half) * kPlane + l16 * RP + 4 * g;
    for (int turn = 0; turn < 2; ++turn) {
        if ((wave >= half) == (turn == 0)) {
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                v4f* p = (v4f*)(mine + 16 * r);
                *p = turn == 0 ? acc[r] : acc[r] + *p;
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
// sum of shrink's parts in order, as an operand in registers.  Steps of 64 columns,
// four MFMA tiles; the matrix goes through LDS and so do the products, so that every
// load and store has neighbouring lanes side by side in a row.  Memory bounds it: 4096
// rows -> 21504, rank 64, 94 us (3.8 TB/s; a plain copy by the same tiles and steps 77),
// 8192 rows -> 4096, rank 32, 36 us (3.7 TB/s).
template <class Frag, int RT, int OUT>
struct ExpandForm {
    static constexpr int KC = (RT + 1) / 2, ranks = 32 * KC;  // steps of 32 ranks
    static constexpr int parts = Frag::bf16 ? 3 : 1;
    static constexpr int PT = 4, step = 16 * PT;
    // base and out go by units of 16 bytes, `lanes` of them a row of a step
    static constexpr int values = OUT == DT_BF16 ? 8 : 4, lanes = step / values, units = 16 * lanes / 64;
    static __device__ __forceinline__ int unit_row(int u) { return u * (64 / lanes) + (threadIdx.x & 63) / lanes; }
    static __device__ __forceinline__ int unit_column() { return values * (threadIdx.x & (lanes - 1)); }
};

// The products of 16 rows of a step in LDS on their way from MFMA's layout.
constexpr int kSumsPitch = 68;  // sixteen rows' writes and reads meet no bank twice
constexpr int kSums = 16 * kSumsPitch;

// A step's part of the matrix in LDS: [C][rank] by column, pitch chosen so that
// sixteen columns' reads meet no bank twice; [rank][C] (backward) as it is for bf16,
// which reads it transposing, and by column for f32.
template <class Frag, int RT, bool COLS>
struct ExpandBlock {
    static constexpr int ranks = 32 * ((RT + 1) / 2);
    static constexpr bool by_rank = Frag::bf16 && !COLS;
    static constexpr int pitch = by_rank ? 64 : Frag::bf16 ? ranks + 8 : ranks + 4;
    static constexpr int bytes = (by_rank ? ranks : 64) * pitch * (Frag::bf16 ? 2 : 4);
};

// A unit of a row from value `at` on, the first n of its values.
template <int DT>
__device__ __forceinline__ v4u unit_load(const void* p, int64_t at, int n) {
    if constexpr (DT == DT_BF16) {
        const uint16_t* q = (const uint16_t*)p + at;
        if (n >= 8) return *(const v4u*)q;
        uint32_t u[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = i < n ? q[i] : 0u;
        return v4u{u[0] | (u[1] << 16), u[2] | (u[3] << 16), u[4] | (u[5] << 16), u[6] | (u[7] << 16)};
    } else {
        const uint32_t* q = (const uint32_t*)p + at;
        if (n >= 4) return *(const v4u*)q;
        return v4u{n > 0 ? q[0] : 0u, n > 1 ? q[1] : 0u, n > 2 ? q[2] : 0u, 0u};
    }
}

template <int DT>
__device__ __forceinline__ void unit_store(void* p, int64_t at, int n, v4u v) {
    if constexpr (DT == DT_BF16) {
        uint16_t* q = (uint16_t*)p + at;
        if (n >= 8) {
            *(v4u*)q = v;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n) q[i] = (uint16_t)(v[i >> 1] >> (16 * (i & 1)));
        }
    } else {
        uint32_t* q = (uint32_t*)p + at;
        if (n >= 4) {
            *(v4u*)q = v;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < n) q[i] = v[i];
        }
    }
}

// Row `row`'s low-rank values, the lane's ranks 8 (lane / 16) .. of each 32, as
// operands; `writes`: to h_out as well.
template <class Frag, int PARTS, int RT>
__device__ __forceinline__ void lora_values(const LoraArgs& a, int row, float scale, bool writes,
                                            Frag (&h)[(RT + 1) / 2][PARTS]) {
    constexpr int RP = 16 * RT, kAhead = 4;
    const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int q = 0; q < (RT + 1) / 2; ++q) {
        const int rank = 32 * q + 8 * g;
        const float* p = a.part + (int64_t)row * RP + rank;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
        if (rank < RP) {
            for (int s0 = 0; s0 < a.splits; s0 += kAhead) {
                float t[kAhead][8];
#pragma unroll
                for (int u = 0; u < kAhead; ++u)
                    if (s0 + u < a.splits) __builtin_memcpy(t[u], p + (int64_t)(s0 + u) * a.m * RP, 32);
#pragma unroll
                for (int u = 0; u < kAhead; ++u)
                    if (s0 + u < a.splits) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = s0 + u == 0 ? t[u][i] : v[i] + t[u][i];
                    }
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (rank + i < a.rank) {
                if (writes) a.h_out[(int64_t)row * a.rank + rank + i] = v[i];
                v[i] *= scale;
            } else {
                v[i] = 0.0f;
            }
        }
        if constexpr (Frag::bf16) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t parts[3];
                bf16_parts(v[2 * i], v[2 * i + 1], parts);
#pragma unroll
                for (int s = 0; s < PARTS; ++s) h[q][s].v[i] = (int)parts[s];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) h[q][0].v[i] = v[i];
        }
    }
}

// 16 rows of a step: the lanes' base units plus the products, stored (WHOLE: no row
// or column of the step is missing, or a row's stand-in has the same results).
template <class F, int OUT, bool WHOLE>
__device__ __forceinline__ void lora_store(const LoraArgs& a, const int64_t (&at)[F::units], int count, int c,
                                           v4u (&x)[F::units], const v4f (&acc)[F::PT], float* sums) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int p = 0; p < F::PT; ++p) *(v4f*)(sums + (lane & 15) * kSumsPitch + 16 * p + 4 * (lane >> 4)) = acc[p];
    asm volatile("" ::: "memory");  // a wave's LDS accesses go in order
#pragma unroll
    for (int u = 0; u < F::units; ++u) {
        const float* s = sums + F::unit_row(u) * kSumsPitch + F::unit_column();
        if constexpr (OUT == DT_BF16) {
            const v4f lo = *(const v4f*)s, hi = *(const v4f*)(s + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                x[u][i] = f32x2_to_bf16x2(f32_from_bits(x[u][i] << 16) + (i < 2 ? lo[2 * i] : hi[2 * i - 4]),
                                          f32_from_bits(x[u][i] & 0xffff0000u) + (i < 2 ? lo[2 * i + 1] : hi[2 * i - 3]));
        } else {
            const v4f v = *(const v4f*)s;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[u][i] = f32_bits(f32_from_bits(x[u][i]) + v[i]);
        }
    }
    asm volatile("" ::: "memory");
    const int first = c + F::unit_column();
#pragma unroll
    for (int u = 0; u < F::units; ++u) {
        if constexpr (WHOLE) unit_store<OUT>(a.out, at[u] + first, 64, x[u]);
        else if (F::unit_row(u) < count && first < a.C) unit_store<OUT>(a.out, at[u] + first, a.C - first, x[u]);
    }
}

template <class F, int OUT>
__device__ __forceinline__ void lora_base(const LoraArgs& a, const int64_t (&at)[F::units], int count, int c,
                                          v4u (&x)[F::units]) {
    const int first = c + F::unit_column();
#pragma unroll
    for (int u = 0; u < F::units; ++u) {
        x[u] = v4u{0, 0, 0, 0};
        if (a.base && F::unit_row(u) < count && first < a.C) x[u] = unit_load<OUT>(a.base, at[u] + first, a.C - first);
    }
}

// The part of the matrix of a step from memory to LDS, an eight of values at a time: where a thread's come from, and where they go.
template <class Frag, int RT, bool COLS>
struct ExpandLoader {
    using B = ExpandBlock<Frag, RT, COLS>;
    static constexpr int per = B::ranks * 64 / 8 / 256;
    int from[per], to[per], col[per];  // from: values past the step's first, of [rank][C] the rank; -1: none
    int64_t matrix;
    bool whole;

    __device__ __forceinline__ void init(const LoraArgs& a, int64_t first) {
        matrix = first;
        whole = a.rank % 8 == 0;
        const int each = COLS ? (a.rank + 7) / 8 : 8;  // eights of a column's ranks, or of a rank's columns
#pragma unroll
        for (int i = 0; i < per; ++i) {
            const int e = threadIdx.x + 256 * i, major = e / each, minor = 8 * (e - major * each);
            const bool there = COLS ? major < 64 : major < a.rank;
            col[i] = COLS ? major : minor;
            from[i] = there ? (COLS ? major * a.rank + minor : major) : -1;
            to[i] = B::by_rank || COLS ? major * B::pitch + minor : minor * B::pitch + major;
        }
    }

    // WHOLE: all of the step's columns are there and the rank is a multiple of eight;
    // without a branch (a thread without an eight loads the first, which goes nowhere)
    template <bool WHOLE>
    __device__ __forceinline__ void load(const LoraArgs& a, int c, Frag (&raw)[per]) const {
#pragma unroll
        for (int i = 0; i < per; ++i) {
            const int f = max(from[i], 0);
            if constexpr (COLS) {
                const int64_t p = matrix + (int64_t)c * a.rank + f;
                if (!WHOLE && c + col[i] >= a.C) clear(raw[i]);
                else if (WHOLE || whole) load8(a.w, p, a.w_dtype, raw[i]);
                else load8(a.w, p, 1, a.w_dtype, from[i] < 0 ? 0 : a.rank - (f - col[i] * a.rank), raw[i]);
            } else {
                const int64_t p = matrix + (int64_t)f * a.C + c + col[i];
                if (WHOLE || c + col[i] + 8 <= a.C) load8(a.w, p, a.w_dtype, raw[i]);
                else load8(a.w, p, 1, a.w_dtype, a.C - c - col[i], raw[i]);
            }
        }
    }

    __device__ __forceinline__ void put(uint8_t* block, const Frag (&raw)[per]) const {
#pragma unroll
        for (int i = 0; i < per; ++i) {
            if (from[i] < 0) continue;
            if constexpr (Frag::bf16) {
                *(v4i*)((uint16_t*)block + to[i]) = raw[i].v;
            } else if constexpr (COLS) {
                *(float4*)((float*)block + to[i]) = make_float4(raw[i].v[0], raw[i].v[1], raw[i].v[2], raw[i].v[3]);
                *(float4*)((float*)block + to[i] + 4) = make_float4(raw[i].v[4], raw[i].v[5], raw[i].v[6], raw[i].v[7]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) ((float*)block)[to[i] + j * B::pitch] = raw[i].v[j];
            }
        }
    }
};

// acc: 16 rows' low-rank values times a step's part of the matrix.
template <class Frag, int RT, bool COLS, class F>
__device__ __forceinline__ void lora_products(const uint8_t* block, const Frag (&h)[F::KC][F::parts], v4f (&acc)[F::PT]) {
    using B = ExpandBlock<Frag, RT, COLS>;
    const int lane = threadIdx.x & 63, g = lane >> 4, l16 = lane & 15;
#pragma unroll
    for (int p = 0; p < F::PT; ++p) {
        Frag w[F::KC];
#pragma unroll
        for (int q = 0; q < F::KC; ++q) {
            if constexpr (B::by_rank) {
                load_rows((const uint16_t*)block + 32 * q * B::pitch, B::pitch, [&](int i) { return 16 * p + i; }, w[q]);
            } else if constexpr (Frag::bf16) {
                w[q].v = *(const v4i*)((const uint16_t*)block + (16 * p + l16) * B::pitch + 32 * q + 8 * g);
            } else {
                const float* s = (const float*)block + (16 * p + l16) * B::pitch + 32 * q + 8 * g;
                *(float4*)&w[q].v[0] = *(const float4*)s;
                *(float4*)&w[q].v[4] = *(const float4*)(s + 4);
            }
        }
        acc[p] = mma_parts(w, h);
    }
}

// A few rows (at most 16, forward): the waves take every fourth step, each its own
// part of the matrix straight into registers, a step ahead (through LDS 48 rows of
// their own adapters, 4096 -> 16384, rank 16, took 10.8 us for 9.7).
template <class Frag, int OUT, int RT>
__device__ __forceinline__ void lora_expand_few(const LoraArgs& a, const int* rows, int count, int adapter, float* sums) {
    using F = ExpandForm<Frag, RT, OUT>;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, l16 = lane & 15;
    const int c0 = (int)min((int64_t)a.C, (int64_t)blockIdx.y * a.columns) + F::step * wave;
    const int c1 = (int)min((int64_t)a.C, (int64_t)(blockIdx.y + 1) * a.columns);
    if (c0 >= c1) return;  // uniform in the wave
    const int64_t matrix = (int64_t)adapter * a.rank * a.C;
    int64_t at[F::units];
#pragma unroll
    for (int u = 0; u < F::units; ++u) at[u] = (int64_t)rows[min(F::unit_row(u), count - 1)] * a.C;
    const bool whole = a.rank % 8 == 0;
    Frag w[F::PT][F::KC];
    auto load_w = [&](int c) {
#pragma unroll
        for (int p = 0; p < F::PT; ++p) {
            const int64_t from = matrix + (int64_t)min(c + 16 * p + l16, a.C - 1) * a.rank;
#pragma unroll
            for (int q = 0; q < F::KC; ++q) {
                const int rank = 32 * q + 8 * g;
                if (!whole) load8(a.w, from + rank, 1, a.w_dtype, a.rank - rank, w[p][q]);
                else if (rank < a.rank) load8(a.w, from + rank, a.w_dtype, w[p][q]);
                else clear(w[p][q]);
            }
        }
    };
    load_w(c0);
    v4u base[F::units];
    lora_base<F, OUT>(a, at, count, c0, base);
    Frag h[F::KC][F::parts];
    lora_values<Frag, F::parts, RT>(a, rows[min(l16, count - 1)], a.scales ? a.scales[adapter] : 1.0f,
                                    blockIdx.y == 0 && wave == 0 && a.h_out && l16 < count, h);
    for (int c = c0; c < c1; c += 4 * F::step) {
        v4f acc[F::PT];
#pragma unroll
        for (int p = 0; p < F::PT; ++p) acc[p] = mma_parts(w[p], h);
        v4u x[F::units];
#pragma unroll
        for (int u = 0; u < F::units; ++u) x[u] = base[u];
        if (c + 4 * F::step < c1) {
            load_w(c + 4 * F::step);
            lora_base<F, OUT>(a, at, count, c + 4 * F::step, base);
        }
        lora_store<F, OUT, false>(a, at, count, c, x, acc, sums);
    }
}

// Columns [c0, c1) of a tile of the plan: 16 rows per wave, every wave the same
// columns.  The step's part of the matrix is in one of two buffers in LDS; those of
// the next `ahead` steps are on their way, as is their base (loads come back in order:
// waiting for a younger part of the matrix waits for every older base).
template <class Frag, int OUT, int RT, bool COLS>
__device__ __forceinline__ void lora_expand_tile(const LoraArgs& a, const int* rows, int count, int adapter, int c0, int c1,
                                                 uint8_t* lds, float* sums) {
    using F = ExpandForm<Frag, RT, OUT>;
    using B = ExpandBlock<Frag, RT, COLS>;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15;
    const int own = 16 * wave, left = min(16, count - own);  // the wave's rows
    int64_t at[F::units];
#pragma unroll
    for (int u = 0; u < F::units; ++u) at[u] = (int64_t)rows[min(own + F::unit_row(u), count - 1)] * a.C;
    using L = ExpandLoader<Frag, RT, COLS>;
    L w;
    w.init(a, (int64_t)adapter * a.rank * a.C);
    Frag h[F::KC][F::parts];
    const float scale = a.scales ? a.scales[adapter] : 1.0f;
    // ranks past the last stay zero in both buffers
    for (int i = 16 * threadIdx.x; i < 2 * B::bytes; i += 16 * 256) *(v4i*)(lds + i) = v4i{0, 0, 0, 0};
    // Whole steps without a branch, so that the counts of loads in flight are known and
    // a wait for one load waits for no store: a row past the tile's is its last one
    // again, with the same results (and where a step ahead is none, the last one again).
    // A rank that is no multiple of eight takes the other columns' way.
    const int steps = !COLS || w.whole ? (min(c1, a.C / F::step * F::step) - c0) / F::step : 0;
    auto run = [&](auto based) {
        constexpr int D = RT <= 2 && Frag::bf16 ? 4 : RT <= 4 ? 3 : 2;  // what the registers hold
        v4u base[D][F::units];
        Frag raw[D][L::per];
        auto load_base = [&](int step, v4u (&x)[F::units]) {
            const int c = c0 + min(step, steps - 1) * F::step + F::unit_column();
#pragma unroll
            for (int u = 0; u < F::units; ++u) {
                x[u] = v4u{0, 0, 0, 0};
                if constexpr (based.value) x[u] = unit_load<OUT>(a.base, at[u] + c, 64);
            }
        };
        auto ahead_w = [&](int step, Frag (&r)[L::per]) { w.template load<true>(a, c0 + min(step, steps - 1) * F::step, r); };
#pragma unroll
        for (int d = 0; d < D; ++d) {
            ahead_w(d, raw[d]);
            load_base(d, base[d]);
        }
        lora_values<Frag, F::parts, RT>(a, rows[min(own + l16, count - 1)], scale, c0 == 0 && a.h_out && l16 < left, h);
        __syncthreads();
        w.put(lds, raw[0]);
        ahead_w(D, raw[0]);
        __syncthreads();
        for (int s0 = 0; s0 < steps; s0 += D) {
#pragma unroll
            for (int d = 0; d < D; ++d) {
                const int step = s0 + d, turn = step & 1;
                if (step >= steps) break;  // uniform
                w.put(lds + (turn ^ 1) * B::bytes, raw[(d + 1) % D]);
                ahead_w(step + 1 + D, raw[(d + 1) % D]);
                v4u x[F::units];
#pragma unroll
                for (int u = 0; u < F::units; ++u) x[u] = base[d][u];
                load_base(step + D, base[d]);
                __builtin_amdgcn_sched_barrier(0);  // the loads ahead of the products
                v4f acc[F::PT];
                lora_products<Frag, RT, COLS, F>(lds + turn * B::bytes, h, acc);
                if (left > 0) lora_store<F, OUT, true>(a, at, left, c0 + step * F::step, x, acc, sums);  // uniform in the wave
                lds_publish();
            }
        }
    };
    if (steps > 0) {
        if (a.base) run(Yes{});
        else run(No{});
    } else {
        lora_values<Frag, F::parts, RT>(a, rows[min(own + l16, count - 1)], scale, c0 == 0 && a.h_out && l16 < left, h);
    }
    for (int c = c0 + steps * F::step; c < c1; c += F::step) {  // uniform
        Frag raw[L::per];
        w.template load<false>(a, c, raw);
        v4u x[F::units];
        lora_base<F, OUT>(a, at, left, c, x);
        __syncthreads();
        w.put(lds, raw);
        __syncthreads();
        v4f acc[F::PT];
        lora_products<Frag, RT, COLS, F>(lds, h, acc);
        lora_store<F, OUT, false>(a, at, left, c, x, acc, sums);
    }
}

// Rows without an adapter: columns [c0, c1) of their base.
__device__ __forceinline__ void lora_bare(const LoraArgs& a, const int* rows, int count, int c0, int c1) {
    if (c0 == 0 && a.h_out)
        for (int i = threadIdx.x; i < count * a.rank; i += blockDim.x)
            a.h_out[(int64_t)rows[i / a.rank] * a.rank + i % a.rank] = 0.0f;
    if (a.base == a.out) return;
    // 16 bytes at a time as they are, eight rows in flight a thread; row ends value by value
    const int size = a.out_dtype == DT_BF16 ? 2 : 4, per = 16 / size, wide = (c1 - c0) / per;
    for (int i = threadIdx.x; i < (count + 7) / 8 * wide; i += blockDim.x) {
        const int r0 = i / wide * 8, c = c0 + i % wide * per;
        v4u v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            v[u] = v4u{0, 0, 0, 0};
            if (a.base && r0 + u < count) v[u] = *(const v4u*)((const uint8_t*)a.base + ((int64_t)rows[r0 + u] * a.C + c) * size);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (r0 + u < count) *(v4u*)((uint8_t*)a.out + ((int64_t)rows[r0 + u] * a.C + c) * size) = v[u];
    }
    const int done = c0 + wide * per, rest = c1 - done;
    for (int i = threadIdx.x; i < count * rest; i += blockDim.x) {
        const int64_t at = (int64_t)rows[i / rest] * a.C + done + i % rest;
        store_out(a.out, at, a.base ? load_as_f32(a.base, at, a.out_dtype) : 0.0f, a.out_dtype);
    }
}

// A few rows: a workgroup per leading row and `columns` columns.  The plan's tiles:
// the steps of all tiles, one tile after the other, in as many equal shares as there
// are workgroups (two a CU), so that however the rows fall onto adapters no CU has
// more to do than another, and low-rank values are laid out once or twice by each.
template <class Frag, bool FEW, int RT, bool COLS>
__device__ __forceinline__ void lora_expand(const LoraArgs& a) {
    const int wave = threadIdx.x >> 6;
    __shared__ __align__(16) float sums[4][kSums];
    if constexpr (FEW) {
        __shared__ int rows[16];
        int adapter;
        const int count = lora_few(a, blockIdx.x, rows, adapter);
        if (count == 0) return;  // uniform
        if (adapter == a.adapters)
            lora_bare(a, rows, count, (int)min((int64_t)a.C, (int64_t)blockIdx.y * a.columns),
                      (int)min((int64_t)a.C, (int64_t)(blockIdx.y + 1) * a.columns));
        else if (a.out_dtype == DT_BF16) lora_expand_few<Frag, DT_BF16, RT>(a, rows, count, adapter, sums[wave]);
        else lora_expand_few<Frag, DT_F32, RT>(a, rows, count, adapter, sums[wave]);
    } else {
        __shared__ int rows[kTileRows];
        __shared__ __align__(16) uint8_t lds[2 * ExpandBlock<Frag, RT, COLS>::bytes];
        constexpr int step = 64;
        const int lane = threadIdx.x & 63, per = (a.C + step - 1) / step;
        const int64_t steps = (int64_t)a.counts[0] * per;
        const int share = xcd_order(blockIdx.x, gridDim.x);
        int64_t at = steps * share / gridDim.x;
        const int64_t end = steps * (share + 1) / gridDim.x;
        while (at < end) {  // uniform
            const int tile = (int)(at / per), first = (int)(at - (int64_t)tile * per);
            const int many = (int)min(end - at, (int64_t)(per - first));
            const int adapter = a.tile_adapter[tile];
            const int row = a.slot_row[(int64_t)tile * kTileRows + lane];  // those without a row are the last
            __syncthreads();  // the tile before is done with
            if (threadIdx.x < 64) rows[lane] = row;
            __syncthreads();
            const int count = __popcll(__ballot(row >= 0)), c0 = first * step, c1 = min(a.C, c0 + many * step);
            if (adapter == a.adapters) lora_bare(a, rows, count, c0, c1);
            else if (a.out_dtype == DT_BF16) lora_expand_tile<Frag, DT_BF16, RT, COLS>(a, rows, count, adapter, c0, c1, lds, sums[wave]);
            else lora_expand_tile<Frag, DT_F32, RT, COLS>(a, rows, count, adapter, c0, c1, lds, sums[wave]);
            at += many;
        }
    }
}

// ---- outer ---------------------------------------------------------------------
// grad(rank, c) of an adapter = sum over its rows of ht[rank][slot] x[row][c].  An
// item of the plan is some of an adapter's tiles; one that has them all writes the
// gradient, the others a partial sum each.  A wave has 64 columns, 32 rows a step,
// which bf16 takes through LDS; the next step's rows are on their way meanwhile.
// Workgroups from the grid's end on write the zeros of adapters without rows.
// Both sides of 8192 x 4096, rank 32: 42 us (134 MB of rows read once, 3.2 TB/s).
template <class Frag, int RT, bool COLS>
__device__ __forceinline__ void lora_outer(const LoraArgs& a, int number, int numbers, uint16_t* blocks) {
    constexpr int PARTS = Frag::bf16 ? 3 : 1, CT = 4;
    const int other = numbers - 1 - number;
    if (other < a.adapters && !a.accumulate && a.per_adapter[2 * other] == 0) {
        const int64_t size = (int64_t)a.rank * a.C, share = (int64_t)a.rank * 256;  // this workgroup's columns' worth
        const int64_t from = blockIdx.x * share, to = min(size, from + share);
        for (int64_t i = from + threadIdx.x; i < to; i += 256) a.grad[other * size + i] = 0.0f;
    }
    if (number >= a.counts[1]) return;
    const int32_t* item = a.items + 4 * number;
    const int adapter = item[0], tile = item[1], tiles = item[2], partial = item[3];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, l16 = lane & 15;
    const int64_t first = ((int64_t)blockIdx.x * 4 + wave) * 16 * CT;
    if (first >= a.C) return;
    const int c0 = (int)first;
    v4f acc[CT][RT];
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
    auto sum = [&](auto careful) {
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int r = 0; r < RT; ++r) acc[c][r] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (Frag::bf16) load_rows32(s0);
        for (int64_t s = s0; s < s1; s += 32) {
            const int64_t at = s + 8 * g;
            Frag x[CT], h[RT][PARTS];
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int p = 0; p < PARTS; ++p)
                    load8(a.ht, ((s / 32 * PARTS + p) * RT + r) * 512 + 8 * lane, DT_F32, h[r][p]);
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
            for (int c = 0; c < CT; ++c) {
                Frag rest = x[c];
                if constexpr (careful.value) rest = finite_values(x[c]);
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int p = PARTS - 1; p >= 0; --p) {
                        const Frag& v = p == 0 ? x[c] : rest;
                        acc[c][r] = COLS ? mma(h[r][p], v, acc[c][r]) : mma(v, h[r][p], acc[c][r]);
                    }
            }
        }
    };
    sum(No{});
    if constexpr (Frag::bf16) {  // a sum that is not finite: again, with what is not finite in the first parts' products alone
        bool fine = true;
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i) fine &= __builtin_isfinite(acc[c][r][i]);
        if (__ballot(!fine)) sum(Yes{});  // uniform
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
// again.  Then tiles, and items of up to item_tiles of them.  One CU's instructions
// bound it: 300 rows 4.2 us, 4096 8.7, 8192 11.2, where two launches of many workgroups
// would start twice; past those, with the calls around it, 16384 rows 49 of mixed ids and
// 29 in runs, 49152 115 and 58.
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
    // the lanes of the same adapter
    auto match = [&](int e) {
        uint64_t same = __ballot(e >= 0);
        if (__ballot(e == __builtin_amdgcn_readfirstlane(e)) == ~0ull) return same;  // a run of rows
        for (int b = 0; b < bits; ++b) {
            const uint64_t bal = __ballot(e >= 0 && ((e >> b) & 1));
            same &= ((e >> b) & 1) ? bal : ~bal;
        }
        return same;
    };
    // the row's rank among the wave's rows of its adapter so far, or (counted before) its slot
    auto place = [&](int e) {
        const uint64_t same = match(e);
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
    if (held) {  // as place, every round's addition on its way before the first is waited for
        int leader[kHeld], at[kHeld];
#pragma unroll
        for (int u = 0; u < kHeld; ++u) {
            leader[u] = at[u] = rank[u] = 0;
            if (64 * u >= per) continue;  // uniform
            const uint64_t same = match(e[u]);
            leader[u] = e[u] >= 0 ? __ffsll((unsigned long long)same) - 1 : 0;
            rank[u] = __popcll(same & ((1ull << lane) - 1));
            if (e[u] >= 0 && lane == leader[u]) at[u] = atomicAdd(&mine[e[u]], __popcll(same));
        }
#pragma unroll
        for (int u = 0; u < kHeld; ++u)
            if (64 * u < per) rank[u] += __shfl(at[u], leader[u], kWave);
    } else {
        for (int r = r0; r < r1; r += 64) place(group(r + lane));
    }
    __syncthreads();
    for (int i = tid >> 4; i < G; i += 64) {  // 16 lanes a group: a wave's rows each
        const int w = tid & 15, n = plan_lds[w * G + i];
        int sum = n;
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) {
            const int t = __shfl_up(sum, off, 16);
            if (w >= off) sum += t;
        }
        plan_lds[w * G + i] = sum - n;
        if (w == 15) total[i] = sum;
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

// The low-rank values for the outer products: h as given or the sum of shrink's
// parts, times the adapter's scale, zeros where there is no row or rank; as operands
// whose K runs over slots: per 32 slots, part and 16 ranks the eight values of each
// lane of a wave, so that a wave loads them in one piece.  A tile per workgroup, 16
// ranks at a time turned in LDS.
namespace {

__device__ __forceinline__ void lora_finish(const LoraArgs& a, int r0, float (&turned)[16][kTileRows + 1]) {
    const int tile = blockIdx.x;
    if (tile >= a.counts[0]) return;
    const int adapter = a.tile_adapter[tile];
    if (adapter == a.adapters) return;
    const float scale = a.scales ? a.scales[adapter] : 1.0f;
    const int slot = threadIdx.x >> 2, r4 = 4 * (threadIdx.x & 3), row = a.slot_row[(int64_t)tile * kTileRows + slot];
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
    // four slots of a rank: lane 16 (slot / 8) + rank of the operand of 32 slots
    const int rank = threadIdx.x >> 4, s4 = 4 * (threadIdx.x & 15);
    const int64_t block = (int64_t)tile * 2 + (s4 >> 5), tiles = a.rank_pad / 16;
    const int in = ((s4 >> 3 & 3) * 16 + rank) * 8 + (s4 & 7);
    float u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = turned[rank][s4 + i];
    if (a.x_dtype == DT_BF16) {
        uint32_t lo[3], hi[3];
        bf16_parts(u[0], u[1], lo);
        bf16_parts(u[2], u[3], hi);
#pragma unroll
        for (int q = 0; q < 3; ++q)
            *(uint2*)((uint16_t*)a.ht + ((block * 3 + q) * tiles + r0 / 16) * 512 + in) = make_uint2(lo[q], hi[q]);
    } else {
        *(float4*)((float*)a.ht + (block * tiles + r0 / 16) * 512 + in) = make_float4(u[0], u[1], u[2], u[3]);
    }
}

// An adapter's partial sums in order (8192 x 4096, rank 32, both: 8.4 us).
__device__ __forceinline__ void lora_reduce(const LoraArgs& a, int adapter) {
    const int items = a.per_adapter[2 * adapter];
    if (items < 2) return;
    const int64_t size = (int64_t)a.rank * a.C, i = 4 * ((int64_t)blockIdx.x * 256 + threadIdx.x);
    if (i >= size) return;
    float* to = a.grad + adapter * size + i;
    const float* p = a.gpart + (int64_t)a.per_adapter[2 * adapter + 1] * size + i;
    if (i + 4 <= size) {
        v4f v = {0.0f, 0.0f, 0.0f, 0.0f};
        constexpr int kAhead = 8;
        for (int s0 = 0; s0 < items; s0 += kAhead) {
            v4f t[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (s0 + u < items) __builtin_memcpy(&t[u], p + (s0 + u) * size, 16);
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (s0 + u < items) v += t[u];
        }
        if (a.accumulate) {
            v4f old;
            __builtin_memcpy(&old, to, 16);
            v += old;
        }
        __builtin_memcpy(to, &v, 16);
    } else {
        for (int j = 0; i + j < size; ++j) {
            float v = 0.0f;
            for (int s = 0; s < items; ++s) v += p[s * size + j];
            to[j] = a.accumulate ? to[j] + v : v;
        }
    }
}

// Which of the two a workgroup is for, and its number among that one's.
__device__ __forceinline__ bool lora_second(const LoraPairArgs& p, int& number) {
    number = p.many == 2 ? blockIdx.y >> 1 : blockIdx.y;
    return (p.many == 2 ? blockIdx.y & 1 : p.first) != 0;
}

}  // namespace

extern "C" __global__ __launch_bounds__(256) void nh_lora_finish_kernel(LoraPairArgs p) {
    __shared__ float turned[16][kTileRows + 1];
    int number;
    if (lora_second(p, number)) lora_finish(p.v[1], 16 * number, turned);
    else lora_finish(p.v[0], 16 * number, turned);
}

extern "C" __global__ __launch_bounds__(256) void nh_lora_reduce_kernel(LoraPairArgs p) {
    int number;
    if (lora_second(p, number)) lora_reduce(p.v[1], number);
    else lora_reduce(p.v[0], number);
}

// Compute kind (bf16, or f32 whatever the operands), a few rows or the plan's tiles
// forward, or the plan's backward (matrices the other way), ranks to 16, 32, 64, 128.
#define NH_LORA_RANKS(call, ...) call(__VA_ARGS__, 1) call(__VA_ARGS__, 2) call(__VA_ARGS__, 4) call(__VA_ARGS__, 8)
#define NH_CALL(kind, Frag, rows, FEW, BACK, RT)                                                                     \
    extern "C" __global__ __launch_bounds__(512) void                                                                \
    nh_lora_shrink_##kind##_##rows##_##RT##_kernel(LoraArgs a) {                                                     \
        lora_shrink<Frag, FEW, RT, BACK>(a);                                                                         \
    }                                                                                                                \
    extern "C" __global__ __launch_bounds__(256, RT == 8 ? 1 : 2) void                                               \
    nh_lora_expand_##kind##_##rows##_##RT##_kernel(LoraArgs a) {                                                     \
        lora_expand<Frag, FEW, RT, !BACK>(a);                                                                        \
    }
NH_LORA_RANKS(NH_CALL, bf16, Frag16, few, true, false)
NH_LORA_RANKS(NH_CALL, bf16, Frag16, tiles, false, false)
NH_LORA_RANKS(NH_CALL, bf16, Frag16, back, false, true)
NH_LORA_RANKS(NH_CALL, f32, Frag32, few, true, false)
NH_LORA_RANKS(NH_CALL, f32, Frag32, tiles, false, false)
NH_LORA_RANKS(NH_CALL, f32, Frag32, back, false, true)
#undef NH_CALL
#define NH_CALL(kind, Frag, RT)                                                                                       \
    extern "C" __global__ __launch_bounds__(256) void nh_lora_outer_##kind##_##RT##_kernel(LoraPairArgs p) {          \
        __shared__ __align__(16) uint16_t blocks[Frag::bf16 ? 4 * 32 * 64 : 8];                                      \
        int number;                                                                                                  \
        if (lora_second(p, number)) lora_outer<Frag, RT, true>(p.v[1], number, gridDim.y / p.many, blocks);          \
        else lora_outer<Frag, RT, false>(p.v[0], number, gridDim.y / p.many, blocks);                                \
    }
NH_LORA_RANKS(NH_CALL, bf16, Frag16)
NH_LORA_RANKS(NH_CALL, f32, Frag32)
#undef NH_CALL
#undef NH_LORA_RANKS
