// Device entry points of the low-rank adapters: validate on the host, then enqueue.
#include <algorithm>
#include <cstdint>

#include "../host/adapters_operands.h"

using namespace nh;

namespace {

constexpr size_t kTileRows = 64;  // of the plan
// Rows that need no plan: one ballot sees all of them, and each 16 of an adapter are a
// workgroup's.  Without the plan 1, 16, 48 and 64 rows of 4096 -> 16384 (the last of
// one adapter of rank 64) take 7.4, 8.9, 12.8 and 15.0 us, with it 12.1, 18.8, 25.1
// and 19.1.
constexpr size_t kFewRows = 64;

int rank_form(size_t rank) { return rank <= 16 ? 0 : rank <= 32 ? 1 : rank <= 64 ? 2 : 3; }
size_t rank_pad(size_t rank) { return (size_t)16 << rank_form(rank); }
size_t most_tiles(size_t m, size_t adapters) { return m / kTileRows + std::min(m, adapters + 1); }

// A few rows: the most 16s of rows of an adapter (or of none).
size_t few_units(size_t m, size_t adapters) { return std::min(m, m / 16 + adapters + 1); }

// How shrink cuts C: columns per wave (eight waves a workgroup), and parts, of which
// there is more than one only while the CUs are not all busy.  A wave has 128 columns at
// least.  A few rows are a few workgroups: 16 rows of 21504, rank 64, take 40, 26, 22, 18,
// 17 and 21 us in 1, 2, 4, 8, 16 and 32 parts, one row of 16384, rank 16, 17, 12, 9.9, 9.5,
// 9.8, 9.8.  The plan's tiles gain to 4: 300 rows of 2701 -> 1999 bf16, rank 20, 24, 20, 18
// and 18 in 1, 2, 4 and 8; 1024 rows of 4096, rank 32, 24, 23, 24, 24.
constexpr size_t kShrinkWaves = 8;
struct Split {
    size_t per_wave, parts;
};

Split shrink_split(size_t m, size_t adapters, size_t c) {
    const size_t units = m <= kFewRows ? few_units(m, adapters) : (m + 15) / 16;
    Split s;
    s.parts = std::max<size_t>(1, std::min<size_t>(m <= kFewRows ? 16 : 4, 512 / units));
    s.per_wave = std::max<size_t>(128, ((c + kShrinkWaves * s.parts - 1) / (kShrinkWaves * s.parts) + 31) / 32 * 32);
    s.parts = (c + kShrinkWaves * s.per_wave - 1) / (kShrinkWaves * s.per_wave);
    return s;
}

// Columns that a workgroup of expand takes of a few rows, for about 768 workgroups:
// each sums the low-rank values anew.  With 384, 768 and 1536 workgroups 48 rows of 64
// adapters (4096 -> 16384, rank 16) take 15.6, 12.8 and 14.0 us, 16 rows of them 10.5, 9.7
// and 9.6, 64 rows of one adapter (4096 -> 21504, rank 64) 14.7, 15.8 and 15.8, one row the
// same.
size_t expand_columns(size_t m, size_t adapters, size_t c) {
    const size_t shares = std::max<size_t>(1, 768 / few_units(m, adapters));
    return std::max<size_t>(256, std::min<size_t>(2048, ((c + shares - 1) / shares + 255) / 256 * 256));
}

// Most tiles of an outer item: about 32 items of an evenly dealt batch.  da and db of
// 4096 -> 4096 in 16, 32 and 64 items, us: 4096 rows, rank 32, 53, 57, 71; 8192 rows, rank 8,
// 86, 67, 75, rank 32 97, 83, 100, rank 64 121, 135, 163; 32768 rows, rank 16, 299, 230, 239.
size_t item_tiles(size_t m) { return std::max<size_t>(1, (m / kTileRows + 31) / 32); }

struct Layout {
    size_t slot_row, tile_adapter, counts, items, per_adapter;
    size_t part_x, part_d, ht_h, ht_d, gpart_a, gpart_b;
    size_t slots, items_most, bytes;
};

Layout lora_layout(size_t m, size_t n, size_t k, size_t rank, size_t adapters, bool backward) {
    Layout l{};
    size_t cur = 0;
    auto take = [&](size_t bytes) {
        const size_t o = cur;
        cur += align256(bytes);
        return o;
    };
    const size_t rp = rank_pad(rank), tiles = most_tiles(m, adapters);
    l.slots = tiles * kTileRows;
    if (m > kFewRows || backward) {
        l.slot_row = take(l.slots * 4);
        l.tile_adapter = take(tiles * 4);
        l.counts = take(8);
    }
    l.part_x = take(shrink_split(m, adapters, k).parts * m * rp * 4);
    if (backward) {
        const size_t it = item_tiles(m);
        // of adapters with more than `it` tiles: t / it + 1 < 2 t / it items each, and over 64 it rows, so
        // fewer than 3 per 64 it rows
        const size_t partials = std::min(2 * (tiles / it) + 2, 3 * (m / (kTileRows * it) + 1));
        l.items_most = tiles / it + std::min(m, adapters) + 1;
        l.items = take(l.items_most * 16);
        l.per_adapter = take(adapters * 8);
        l.part_d = take(shrink_split(m, adapters, n).parts * m * rp * 4);
        l.ht_h = take(rp * l.slots * 6);
        l.ht_d = take(rp * l.slots * 6);
        l.gpart_a = take(partials * rank * k * 4);
        l.gpart_b = take(partials * rank * n * 4);
    }
    l.bytes = cur;
    return l;
}

nh_status check_lora(size_t m, size_t n, size_t k, size_t rank, size_t adapters, std::initializer_list<nh_dtype> dtypes,
                     nh_error* err) {
    if (n == 0 || k == 0 || rank == 0 || adapters == 0)
        return set_error(err, NH_INVALID_SHAPE, "invalid adapter shape k=%zu n=%zu rank=%zu adapters=%zu", k, n, rank, adapters);
    if (m == 0) return set_error(err, NH_INVALID_ROW_COUNT, "row_count must be non-zero, got 0");
    for (nh_dtype d : dtypes)
        if (nh_status st = check_dtype(d, err)) return st;
    if (!nh_supports_linear_lora(m, n, k, rank, adapters))
        return set_error(err, NH_UNSUPPORTED, "shape m=%zu n=%zu k=%zu rank=%zu adapters=%zu outside the gfx950 envelope "
                         "(m < 2^24, n and k <= 2^20, m * n and m * k < 2^40, rank <= 128, adapters <= 1024)", m, n, k,
                         rank, adapters);
    return NH_OK;
}

nh_status check_workspace(const void* workspace, size_t given, size_t need, nh_error* err) {
    if (!workspace || given < need) return mismatch(err, "workspace", need, given);
    if (!aligned16(workspace)) return set_error(err, NH_UNSUPPORTED, "workspace must be 16-byte aligned");
    return NH_OK;
}

// One call's launches over its rows.
struct Lora {
    nh_context* ctx;
    nh_stream stream;
    nh_error* err;
    size_t m, rank, adapters;
    bool few;
    LoraArgs common;

    nh_status plan(const Layout& l, uint8_t* ws, const int32_t* ids, bool items) {
        LoraPlanArgs p{};
        p.ids = ids;
        p.slot_row = (int32_t*)(ws + l.slot_row);
        p.tile_adapter = (int32_t*)(ws + l.tile_adapter);
        p.counts = (int32_t*)(ws + l.counts);
        p.items = items ? (int32_t*)(ws + l.items) : nullptr;
        p.per_adapter = items ? (int32_t*)(ws + l.per_adapter) : nullptr;
        p.m = (int)m;
        p.adapters = (int)adapters;
        p.item_tiles = (int)item_tiles(m);
        return launch(ctx, K_LORA_PLAN, 1, 1024, 20 * (adapters + 1) * 4, stream, p, err);
    }

    KernelId form(KernelId first, bool bf16, bool back) const {
        return (KernelId)(first + (bf16 ? 0 : 12) + (few ? 0 : back ? 8 : 4) + rank_form(rank));
    }
    // part = x w^T by parts of C; back: w is [C][rank]
    nh_status shrink(const void* x, nh_dtype xd, const void* w, nh_dtype wd, bool back, size_t c, float* part) {
        LoraArgs a = common;
        const Split s = shrink_split(m, adapters, c);
        a.x = x;
        a.w = w;
        a.part = part;
        a.C = (int)c;
        a.x_dtype = xd;
        a.w_dtype = wd;
        a.per_wave = (int)s.per_wave;
        // a unit of 16 rows a workgroup, in whole turns of the XCDs; half the waves' sums,
        // and before that what lies in LDS to be turned (ShrinkForm of the kernels)
        const size_t units = few ? few_units(m, adapters) : (4 * most_tiles(m, adapters) + 7) / 8 * 8, rp = rank_pad(rank);
        const bool bf16 = xd == NH_BF16 && wd == NH_BF16;
        const size_t turned = !bf16 ? 0 : back ? 16 * 72 + 64 * rp : 3 * 16 * 72;
        const size_t lds = kShrinkWaves * std::max(16 * rp * 2, 2 * turned);
        return launch(ctx, form(K_LORA_SHRINK, bf16, back), (unsigned)units, 64 * (unsigned)kShrinkWaves, lds, stream, a, err,
                      (unsigned)s.parts);
    }

    // out = base + s h w, h the sum of `splits` parts; back: w is [rank][C]
    nh_status expand(const float* part, size_t splits, const void* w, nh_dtype wd, bool back, size_t c, const void* base,
                     void* out, nh_dtype od, float* h_out) {
        LoraArgs a = common;
        a.part = const_cast<float*>(part);
        a.splits = (int)splits;
        a.w = w;
        a.base = base;
        a.out = out;
        a.h_out = h_out;
        a.C = (int)c;
        a.w_dtype = wd;
        a.out_dtype = od;
        const KernelId id = form(K_LORA_EXPAND, wd == NH_BF16, back);
        if (few) {
            const size_t columns = expand_columns(m, adapters, c);
            a.columns = (int)columns;
            return launch(ctx, id, (unsigned)few_units(m, adapters), 256, 0, stream, a, err, (unsigned)((c + columns - 1) / columns));
        }
        // two workgroups a CU, or one per step of 64 columns where there are fewer
        const size_t steps = ((m + kTileRows - 1) / kTileRows + std::min(m, adapters)) * ((c + 63) / 64);
        const size_t shares = std::min<size_t>(2 * (size_t)ctx->cu_count, steps);
        return launch(ctx, id, (unsigned)((shares + 7) / 8 * 8), 256, 0, stream, a, err);
    }

    // The gradients of one or both matrices from the low-rank values that belong to the
    // other side: da from x and dh, db from dout and h.
    struct Gradient {
        const void* x;
        nh_dtype dtype;
        const float *h, *part;  // low-rank values: h as given, or the sum of shrink's parts
        size_t splits, c;
        void* ht;
        float *gpart, *grad;
    };

    nh_status gradients(const Gradient (&g)[2], bool accumulate, size_t items) {
        LoraPairArgs p{};
        for (int i = 0; i < 2; ++i) {
            LoraArgs& a = p.v[i] = common;
            a.h = g[i].h;
            a.part = const_cast<float*>(g[i].part);
            a.splits = (int)g[i].splits;
            a.ht = g[i].ht;
            a.x = g[i].x;
            a.x_dtype = g[i].dtype;
            a.gpart = g[i].gpart;
            a.grad = g[i].grad;
            a.C = (int)g[i].c;
            a.accumulate = accumulate;
        }
        auto launch_pair = [&](KernelId id, int first, int many, size_t gx, size_t gy) {
            p.first = first;
            p.many = many;
            return launch(ctx, id, (unsigned)gx, 256, 0, stream, p, err, (unsigned)(gy * many));
        };
        auto outer_id = [&](int i) { return (KernelId)(K_LORA_OUTER + (g[i].dtype == NH_BF16 ? 0 : 4) + rank_form(rank)); };
        auto columns = [&](int i) { return (g[i].c + 255) / 256; };
        const bool both = g[0].grad && g[1].grad;
        const int first = g[0].grad ? 0 : 1, many = both ? 2 : 1, last = first + many - 1;
        const size_t c = std::max(g[first].c, g[last].c);
        nh_status st = launch_pair(K_LORA_FINISH, first, many, most_tiles(m, adapters), rank_pad(rank) / 16);
        if (st) return st;
        if (both && outer_id(0) != outer_id(1)) {
            if ((st = launch_pair(outer_id(0), 0, 1, columns(0), items)) || (st = launch_pair(outer_id(1), 1, 1, columns(1), items)))
                return st;
        } else if ((st = launch_pair(outer_id(first), first, many, (c + 255) / 256, items))) {
            return st;
        }
        if (m <= kTileRows * item_tiles(m)) return NH_OK;  // one item an adapter
        return launch_pair(K_LORA_REDUCE, first, many, (rank * c + 1023) / 1024, adapters);
    }
};

Lora make_lora(nh_context* ctx, const int32_t* ids, const float* scales, size_t m, size_t rank, size_t adapters,
               bool few, const Layout& l, uint8_t* ws, nh_stream stream, nh_error* err) {
    Lora c{ctx, stream, err, m, rank, adapters, few, {}};
    c.common.ids = ids;
    c.common.scales = scales;
    c.common.slot_row = (int32_t*)(ws + l.slot_row);
    c.common.tile_adapter = (int32_t*)(ws + l.tile_adapter);
    c.common.counts = (int32_t*)(ws + l.counts);
    c.common.items = (int32_t*)(ws + l.items);
    c.common.per_adapter = (int32_t*)(ws + l.per_adapter);
    c.common.m = (int)m;
    c.common.rank = (int)rank;
    c.common.rank_pad = (int)rank_pad(rank);
    c.common.adapters = (int)adapters;
    c.common.numbered = few && few_units(m, adapters) < m;
    return c;
}

}  // namespace

extern "C" {

int nh_supports_linear_lora(size_t m, size_t n, size_t k, size_t rank, size_t adapters) {
    return m > 0 && n > 0 && k > 0 && rank > 0 && adapters > 0 && m < (1u << 24) && n <= (1u << 20) && k <= (1u << 20) &&
           (uint64_t)m * n < (1ull << 40) && (uint64_t)m * k < (1ull << 40) && rank <= 128 && adapters <= 1024;
}

size_t nh_linear_lora_workspace_size(size_t m, size_t n, size_t k, size_t rank, size_t adapters) {
    return nh_supports_linear_lora(m, n, k, rank, adapters) ? lora_layout(m, n, k, rank, adapters, false).bytes : 0;
}

size_t nh_linear_lora_backward_workspace_size(size_t m, size_t n, size_t k, size_t rank, size_t adapters) {
    return nh_supports_linear_lora(m, n, k, rank, adapters) ? lora_layout(m, n, k, rank, adapters, true).bytes : 0;
}

nh_status nh_linear_lora(nh_context* ctx, const void* x, nh_dtype x_dtype, const int32_t* adapter_ids, const void* a,
                         const void* b, nh_dtype w_dtype, const float* scales, size_t m, size_t n, size_t k, size_t rank,
                         size_t adapters, const void* base, void* out, nh_dtype out_dtype, float* h_out,
                         void* workspace, size_t workspace_bytes, nh_stream stream, nh_error* err) {
    clear_error(err);
    nh_status st;
    if ((st = check_lora(m, n, k, rank, adapters, {x_dtype, w_dtype, out_dtype}, err)) ||
        (st = check_given({x, adapter_ids, a, b, out}, err)) ||
        (st = lora_apart(x, x_dtype, adapter_ids, a, b, w_dtype, scales, m, n, k, rank, adapters, base, out, out_dtype, h_out, err)))
        return st;
    const Layout l = lora_layout(m, n, k, rank, adapters, false);
    if ((st = check_workspace(workspace, workspace_bytes, l.bytes, err)) || (st = bind_device(ctx, err))) return st;
    uint8_t* ws = (uint8_t*)workspace;
    Lora c = make_lora(ctx, adapter_ids, scales, m, rank, adapters, m <= kFewRows, l, ws, stream, err);
    float* part = (float*)(ws + l.part_x);
    if (!c.few && (st = c.plan(l, ws, adapter_ids, false))) return st;
    if ((st = c.shrink(x, x_dtype, a, w_dtype, false, k, part))) return st;
    return c.expand(part, shrink_split(m, adapters, k).parts, b, w_dtype, false, n, base, out, out_dtype, h_out);
}

nh_status nh_linear_lora_backward(nh_context* ctx, const void* x, nh_dtype x_dtype, const int32_t* adapter_ids,
                                  const void* a, const void* b, nh_dtype w_dtype, const float* scales, const float* h,
                                  const void* dout, nh_dtype dout_dtype, size_t m, size_t n, size_t k, size_t rank,
                                  size_t adapters, const void* dx_base, void* dx, float* da, float* db, int accumulate,
                                  void* workspace, size_t workspace_bytes, nh_stream stream, nh_error* err) {
    clear_error(err);
    nh_status st;
    if ((st = check_lora(m, n, k, rank, adapters, {x_dtype, w_dtype, dout_dtype}, err)) ||
        (st = check_given({adapter_ids, dout}, err)))
        return st;
    if (!dx && !da && !db) return set_error(err, NH_INVALID_PARAMS, "null operand");
    const bool again = db && !h;  // h is computed here
    if (((da || again) && (st = check_given({x}, err))) || ((dx || again) && (st = check_given({a}, err))) ||
        ((dx || da) && (st = check_given({b}, err))) ||
        (st = lora_backward_apart(x, x_dtype, adapter_ids, a, b, w_dtype, scales, h, dout, dout_dtype, m, n, k, rank, adapters,
                                  dx_base, dx, da, db, err)))
        return st;
    const Layout l = lora_layout(m, n, k, rank, adapters, true);
    if ((st = check_workspace(workspace, workspace_bytes, l.bytes, err)) || (st = bind_device(ctx, err))) return st;
    uint8_t* ws = (uint8_t*)workspace;
    Lora c = make_lora(ctx, adapter_ids, scales, m, rank, adapters, false, l, ws, stream, err);
    float *part_x = (float*)(ws + l.part_x), *part_d = (float*)(ws + l.part_d);
    const size_t parts_x = shrink_split(m, adapters, k).parts, parts_d = shrink_split(m, adapters, n).parts;
    if ((st = c.plan(l, ws, adapter_ids, true))) return st;
    if (again && (st = c.shrink(x, x_dtype, a, w_dtype, false, k, part_x))) return st;
    if ((dx || da) && (st = c.shrink(dout, dout_dtype, b, w_dtype, true, n, part_d))) return st;
    if (dx && (st = c.expand(part_d, parts_d, a, w_dtype, true, k, dx_base, dx, x_dtype, nullptr))) return st;
    if (!da && !db) return NH_OK;
    const Lora::Gradient g[2] = {
        {x, x_dtype, nullptr, part_d, parts_d, k, ws + l.ht_d, (float*)(ws + l.gpart_a), da},
        {dout, dout_dtype, h, part_x, parts_x, n, ws + l.ht_h, (float*)(ws + l.gpart_b), db}};
    return c.gradients(g, accumulate != 0, std::max(l.items_most, adapters));
}

}  // extern "C"
