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
// a token once per eight routes, but for gather with dw, which goes over the rows
// twice (for all dw first, then for out).  One workgroup per token, so that pos and
// the weights are uniform and a weight's gradient is one sum of the workgroup; 16
// bytes of a row per thread and turn, eight routes in flight, as many threads as take
// the row in the fewest turns.  Rows of 64 MiB and more in all go past the caches,
// which they would only sweep.  8192 x 2688 bf16, 6 routes each: dispatch (308 MB)
// 55 us, 74 through the caches; combine (308 MB) 60, with a dispatch of the same rows
// ahead of it 118 and 158 for the two; combine backward with dw (573 MB) 108; dispatch
// backward 59: 5.2 to 5.6 TB/s, the rate of a copy; with dw 92.
// Sums run in f32, over j in route order; results do not change from run to run.
#include "nh_device.h"

using namespace nh;

namespace {

constexpr int kRowRoutes = 8;  // routes in flight

// What a thread has of a row: V consecutive values, as they lie in memory.
template <int DT, int V>
struct RowPart {
    static constexpr int bytes = V * (DT == DT_BF16 ? 2 : 4), words = bytes / 4;
    uint32_t u[words];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < words; ++i) u[i] = 0u;
    }

    __device__ __forceinline__ void load(const void* p, int64_t at) {
        __builtin_memcpy(u, (const uint8_t*)p + at * (bytes / V), bytes);
    }

    // past the caches where `far`
    __device__ __forceinline__ void load(const void* p, int64_t at, bool far) {
        static_assert(bytes == 16, "one load");
        if (!far) return load(p, at);
        typedef uint32_t v4u __attribute__((ext_vector_type(4), aligned(2)));
        const v4u v = __builtin_nontemporal_load((const v4u*)((const uint8_t*)p + at * (bytes / V)));
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = v[i];
    }

    __device__ __forceinline__ float value(int i) const {
        if constexpr (DT == DT_BF16) return f32_from_bits(i & 1 ? u[i >> 1] & 0xffff0000u : u[i >> 1] << 16);
        else return f32_from_bits(u[i]);
    }
};

template <int DT, int V>
__device__ __forceinline__ void row_store(void* p, int64_t at, const float (&v)[V], bool far = false) {
    constexpr int words = DT == DT_BF16 ? V / 2 : V;
    uint32_t x[words];
#pragma unroll
    for (int i = 0; i < words; ++i) {
        if constexpr (DT == DT_BF16) x[i] = f32x2_to_bf16x2(v[2 * i], v[2 * i + 1]);
        else x[i] = f32_bits(v[i]);
    }
    uint8_t* q = (uint8_t*)p + at * (DT == DT_BF16 ? 2 : 4);
    if constexpr (words == 4) {
        typedef uint32_t v4u __attribute__((ext_vector_type(4), aligned(2)));
        if (far) {
            __builtin_nontemporal_store(v4u{x[0], x[1], x[2], x[3]}, (v4u*)q);
            return;
        }
    }
    __builtin_memcpy(q, x, 4 * words);
}

// The routes j0 .. of token t: their slots, and weights; -1 and 0 where there is none.
__device__ __forceinline__ void row_routes(const MoeRowsArgs& a, int64_t t, int j0, int (&slot)[kRowRoutes],
                                           float (&w)[kRowRoutes]) {
    int s[kRowRoutes];
    float given[kRowRoutes];
#pragma unroll
    for (int j = 0; j < kRowRoutes; ++j) s[j] = j0 + j < a.top_k ? a.pos[t * a.top_k + j0 + j] : -1;
#pragma unroll
    for (int j = 0; j < kRowRoutes; ++j) given[j] = a.weights && j0 + j < a.top_k ? a.weights[t * a.top_k + j0 + j] : 1.0f;
#pragma unroll
    for (int j = 0; j < kRowRoutes; ++j) {
        const bool there = s[j] >= 0 && s[j] < a.slots;
        slot[j] = __builtin_amdgcn_readfirstlane(there ? s[j] : -1);
        w[j] = f32_from_bits((uint32_t)__builtin_amdgcn_readfirstlane((int)f32_bits(there ? given[j] : 0.0f)));
    }
}

// The workgroup's sums of d, one per route, to dweights: the wave's eight sums in
// ten lane moves, each of the first three halving how many values a lane has.
__device__ __forceinline__ void row_dweights(const MoeRowsArgs& a, int64_t t, int j0, const float (&d)[kRowRoutes],
                                             float (&red)[16][kRowRoutes]) {
    static_assert(kRowRoutes == 8, "three halvings");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    float v4[4], v2[2], v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v4[i] = (lane & 32 ? d[i + 4] : d[i]) + __shfl_xor(lane & 32 ? d[i] : d[i + 4], 32, kWave);
#pragma unroll
    for (int i = 0; i < 2; ++i) v2[i] = (lane & 16 ? v4[i + 2] : v4[i]) + __shfl_xor(lane & 16 ? v4[i] : v4[i + 2], 16, kWave);
    v = (lane & 8 ? v2[1] : v2[0]) + __shfl_xor(lane & 8 ? v2[0] : v2[1], 8, kWave);
#pragma unroll
    for (int off = 4; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
    if ((lane & 7) == 0) red[wave][(lane >> 5 & 1) * 4 + (lane >> 4 & 1) * 2 + (lane >> 3 & 1)] = v;
    __syncthreads();
    if ((int)threadIdx.x < kRowRoutes && j0 + (int)threadIdx.x < a.top_k) {
        float sum = red[0][threadIdx.x];
        for (int w = 1; w < waves; ++w) sum += red[w][threadIdx.x];
        a.dweights[t * a.top_k + j0 + threadIdx.x] = sum;
    }
    __syncthreads();
}

// d[j] += <rows_in[slot j], v[t]> over the thread's columns [c, c + V), or those of them up to H.
template <int TOKEN, int ROW, int V>
__device__ __forceinline__ void row_dots(const MoeRowsArgs& a, const void* v, int64_t t, int c, const int (&slot)[kRowRoutes],
                                         float (&d)[kRowRoutes]) {
    const int H = a.hidden;
    if (H - c >= V) {
        RowPart<TOKEN, V> x;
        RowPart<ROW, V> y[kRowRoutes];
        x.load(v, t * H + c);
#pragma unroll
        for (int j = 0; j < kRowRoutes; ++j) {
            y[j].clear();
            if (slot[j] >= 0) y[j].load(a.rows_in, (int64_t)slot[j] * H + c, a.far);
        }
#pragma unroll
        for (int j = 0; j < kRowRoutes; ++j)
            if (slot[j] >= 0) {
#pragma unroll
                for (int i = 0; i < V; ++i) d[j] = __builtin_fmaf(y[j].value(i), x.value(i), d[j]);
            }
    } else {
        for (int i = c; i < H; ++i) {
            const float x = load_as_f32(v, t * H + i, TOKEN);
#pragma unroll
            for (int j = 0; j < kRowRoutes; ++j)
                if (slot[j] >= 0) d[j] = __builtin_fmaf(load_as_f32(a.rows_in, (int64_t)slot[j] * H + i, ROW), x, d[j]);
        }
    }
}

template <int TOKEN, int ROW>
__device__ __forceinline__ void scatter_rows(const MoeRowsArgs& a) {
    __shared__ float red[16][kRowRoutes];
    constexpr int V = ROW == DT_BF16 ? 8 : 4;
    const int64_t t = a.token0 + blockIdx.x;
    const int H = a.hidden;
    for (int j0 = 0; j0 < a.top_k; j0 += kRowRoutes) {
        int slot[kRowRoutes];
        float w[kRowRoutes], d[kRowRoutes];
        row_routes(a, t, j0, slot, w);
#pragma unroll
        for (int j = 0; j < kRowRoutes; ++j) d[j] = 0.0f;
        for (uint32_t u = V * threadIdx.x; u < (uint32_t)H; u += V * blockDim.x) {  // u may pass 2^31
            const int c = (int)u;
            // rows_in may be rows_out: the thread's own values, read first
            if (a.dweights) row_dots<TOKEN, ROW, V>(a, a.tokens, t, c, slot, d);
            if (H - c >= V) {
                RowPart<TOKEN, V> v;
                v.load(a.tokens, t * H + c);
#pragma unroll
                for (int j = 0; j < kRowRoutes; ++j)
                    if (slot[j] >= 0) {
                        float o[V];
#pragma unroll
                        for (int i = 0; i < V; ++i) o[i] = w[j] * v.value(i);
                        row_store<ROW, V>(a.rows_out, (int64_t)slot[j] * H + c, o, a.far);
                    }
            } else {
                for (int i = c; i < H; ++i) {
                    const float v = load_as_f32(a.tokens, t * H + i, TOKEN);
#pragma unroll
                    for (int j = 0; j < kRowRoutes; ++j)
                        if (slot[j] >= 0) store_out(a.rows_out, (int64_t)slot[j] * H + i, w[j] * v, ROW);
                }
            }
        }
        if (a.dweights) row_dweights(a, t, j0, d, red);
    }
}

template <int TOKEN, int ROW>
__device__ __forceinline__ void gather_rows(const MoeRowsArgs& a) {
    __shared__ float red[16][kRowRoutes];
    constexpr int V = ROW == DT_BF16 ? 8 : 4;
    const int64_t t = a.token0 + blockIdx.x;
    const int H = a.hidden;
    int slot[kRowRoutes];
    float w[kRowRoutes];
    if (a.dweights) {
        for (int j0 = 0; j0 < a.top_k; j0 += kRowRoutes) {
            float d[kRowRoutes];
            row_routes(a, t, j0, slot, w);
#pragma unroll
            for (int j = 0; j < kRowRoutes; ++j) d[j] = 0.0f;
            for (uint32_t u = V * threadIdx.x; u < (uint32_t)H; u += V * blockDim.x) row_dots<TOKEN, ROW, V>(a, a.dot, t, (int)u, slot, d);
            row_dweights(a, t, j0, d, red);
        }
    }
    row_routes(a, t, 0, slot, w);
    for (uint32_t u = V * threadIdx.x; u < (uint32_t)H; u += V * blockDim.x) {  // u may pass 2^31
        const int c = (int)u;
        float sum[V];
        const bool whole = H - c >= V;
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] = 0.0f;
        if (a.shared) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i < H - c) sum[i] = load_as_f32(a.shared, t * H + c + i, TOKEN);
        }
        for (int j0 = 0; j0 < a.top_k; j0 += kRowRoutes) {
            if (a.top_k > kRowRoutes) row_routes(a, t, j0, slot, w);
            RowPart<ROW, V> y[kRowRoutes];
            if (whole) {
#pragma unroll
                for (int j = 0; j < kRowRoutes; ++j) {
                    y[j].clear();
                    if (slot[j] >= 0) y[j].load(a.rows_in, (int64_t)slot[j] * H + c, a.far);
                }
#pragma unroll
                for (int j = 0; j < kRowRoutes; ++j)
                    if (slot[j] >= 0) {
#pragma unroll
                        for (int i = 0; i < V; ++i) sum[i] = __builtin_fmaf(w[j], y[j].value(i), sum[i]);
                    }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (i < H - c) {
#pragma unroll
                        for (int j = 0; j < kRowRoutes; ++j)
                            if (slot[j] >= 0)
                                sum[i] = __builtin_fmaf(w[j], load_as_f32(a.rows_in, (int64_t)slot[j] * H + c + i, ROW), sum[i]);
                    }
            }
        }
        if (whole) {
            row_store<TOKEN, V>(a.out, t * H + c, sum);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i < H - c) store_out(a.out, t * H + c + i, sum[i], TOKEN);
        }
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

// ---- many routes sorted by expert ----------------------------------------------
// The stable counting sort of nh_moe_permute over chunks of consecutive routes, a
// workgroup each (the last one takes the rest, less than two chunks):
//   count: the chunk's routes per expert, left in the chunk's own part of pos;
//   scan:  one workgroup turns them into each chunk's first slot per expert;
//   place: the chunk's waves take consecutive routes; a wave's 64 routes at a time
//          find their rank among the equal ones by ballots.
// 49152 routes to 128 experts: 4.8 us each alone, 10.5 for the three, 185 in one workgroup.
// pos is its own workspace: a chunk has at least as many routes as there are
// experts, and place has read its part before it writes there.
namespace {

// (Sums of routes may pass 2^31.)
__device__ __forceinline__ void sort_chunk(const MoeSortArgs& a, int c, uint32_t& r0, uint32_t& r1) {
    r0 = (uint32_t)c * a.chunk;
    r1 = c == a.chunks - 1 ? a.routes : r0 + a.chunk;
}

}  // namespace

extern "C" __global__ __launch_bounds__(1024) void nh_moe_sort_count_kernel(MoeSortArgs a) {
    extern __shared__ int sort_lds[];  // [E]
    const int E = a.experts;
    uint32_t r0, r1;
    sort_chunk(a, blockIdx.x, r0, r1);
    for (int e = threadIdx.x; e < E; e += blockDim.x) sort_lds[e] = 0;
    __syncthreads();
    for (uint32_t r = r0 + threadIdx.x; r < r1; r += blockDim.x) {
        const int e = a.indices[r];
        if (e >= 0 && e < E) atomicAdd(&sort_lds[e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += blockDim.x) a.pos[r0 + e] = sort_lds[e];
}

// Threads by expert (up to 1024 at a time) and by part of the chunks.
extern "C" __global__ __launch_bounds__(1024) void nh_moe_sort_scan_kernel(MoeSortArgs a) {
    __shared__ int part[1024], first[1024], wave_sum[16];
    const int E = a.experts, cols = min(E, 1024), parts = 1024 / cols;
    const int col = threadIdx.x % cols, p = threadIdx.x / cols, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int per = (a.chunks + parts - 1) / parts, c0 = min(a.chunks, p * per), c1 = p < parts ? min(a.chunks, c0 + per) : c0;
    int carry = 0;
    for (int base = 0; base < E; base += cols) {
        const int e = base + col;
        constexpr int kAhead = 8;
        int sum = 0;
        if (e < E)
            for (int c = c0; c < c1; c += kAhead) {
                int v[kAhead];
#pragma unroll
                for (int u = 0; u < kAhead; ++u) v[u] = c + u < c1 ? a.pos[(int64_t)(c + u) * a.chunk + e] : 0;
#pragma unroll
                for (int u = 0; u < kAhead; ++u) sum += v[u];
            }
        part[threadIdx.x] = sum;
        __syncthreads();
        int total = 0;  // of expert base + thread
        if ((int)threadIdx.x < cols && base + (int)threadIdx.x < E)
            for (int q = 0; q < parts; ++q) total += part[q * cols + threadIdx.x];
        int incl = total;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int t = __shfl_up(incl, off, kWave);
            if (lane >= off) incl += t;
        }
        if (lane == 63) wave_sum[wave] = incl;
        __syncthreads();
        int before = carry, all = 0;
        for (int w = 0; w < 16; ++w) {
            before += w < wave ? wave_sum[w] : 0;
            all += wave_sum[w];
        }
        if ((int)threadIdx.x < cols && base + (int)threadIdx.x < E) {
            first[threadIdx.x] = before + incl - total;
            a.offsets[base + threadIdx.x] = before + incl - total;
        }
        carry += all;
        __syncthreads();
        if (e < E && p < parts) {
            int at = first[col];
            for (int q = 0; q < p; ++q) at += part[q * cols + col];
            for (int c = c0; c < c1; c += kAhead) {
                int v[kAhead];
#pragma unroll
                for (int u = 0; u < kAhead; ++u) v[u] = c + u < c1 ? a.pos[(int64_t)(c + u) * a.chunk + e] : 0;
#pragma unroll
                for (int u = 0; u < kAhead; ++u)
                    if (c + u < c1) {
                        a.pos[(int64_t)(c + u) * a.chunk + e] = at;
                        at += v[u];
                    }
            }
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) a.offsets[E] = carry;
}

extern "C" __global__ __launch_bounds__(1024) void nh_moe_sort_place_kernel(MoeSortArgs a) {
    extern __shared__ int sort_lds[];  // [waves][E]: the wave's routes per expert, then its next slot
    const int E = a.experts, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    uint32_t c0, c1;
    sort_chunk(a, blockIdx.x, c0, c1);
    const uint32_t per = ((c1 - c0 + waves - 1) / waves + 63) & ~63u;
    const uint32_t r0 = min(c1, c0 + wave * per), r1 = min(c1, r0 + per);
    int* mine = sort_lds + wave * E;
    for (int e = threadIdx.x; e < waves * E; e += blockDim.x) sort_lds[e] = 0;
    __syncthreads();
    for (uint32_t r = r0 + lane; r < r1; r += 64) {
        const int e = a.indices[r];
        if (e >= 0 && e < E) atomicAdd(&mine[e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += blockDim.x) {
        int at = a.pos[c0 + e];
        for (int w = 0; w < waves; ++w) {
            const int n = sort_lds[w * E + e];
            sort_lds[w * E + e] = at;
            at += n;
        }
    }
    __syncthreads();
    int bits = 0;
    while ((1 << bits) < E) ++bits;
    for (uint32_t base = r0; base < r1; base += 64) {  // uniform per wave
        const uint32_t r = base + lane;
        int e = r < r1 ? a.indices[r] : -1;
        if (e >= E) e = -1;
        uint64_t same = __ballot(e >= 0);
        for (int b = 0; b < bits; ++b) {
            const uint64_t bal = __ballot(e >= 0 && ((e >> b) & 1));
            same &= ((e >> b) & 1) ? bal : ~bal;
        }
        const int leader = e >= 0 ? __ffsll((unsigned long long)same) - 1 : 0;
        int slot = 0;
        if (e >= 0 && lane == leader) slot = atomicAdd(&mine[e], __popcll(same));
        slot = __shfl(slot, leader, kWave) + __popcll(same & ((1ull << lane) - 1));
        if (r < r1) a.pos[r] = e >= 0 ? slot : -1;
        if (e >= 0) a.perm[slot] = (int)r;
    }
}
