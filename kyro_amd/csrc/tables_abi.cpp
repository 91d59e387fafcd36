// C ABI of the block tables that live on the GPU (include/kyro_tables.h): argument checks and launches.
#include "kyro_tables.h"

#include <algorithm>
#include <cstdint>

#include "context.hpp"
#include "kernels.hpp"

using namespace kyro::rt;

namespace {

constexpr int kMaxRange = 16;

// Memory of a call, to find arrays that overlap where one of them is written.
struct Ranges {
    struct Range {
        const char* name;
        uintptr_t from, to;
        bool written;
    } r[kMaxRange];
    int n = 0;
    void add(const char* name, const void* p, uint64_t bytes, bool written) {
        if (p && bytes) r[n++] = {name, reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + bytes, written};
    }
    int check(const char* call) const {
        for (int i = 0; i < n; ++i)
            for (int j = 0; j < i; ++j)
                if ((r[i].written || r[j].written) && r[i].from < r[j].to && r[j].from < r[i].to)
                    return fail(KYRO_EINVAL, "%s: %s overlaps %s", call, r[i].name, r[j].name);
        return KYRO_OK;
    }
};

int tables_setup(const kyro_tables_params* p, const char* call, bool extend, const void* state_rows, kyro::TablesArgs& a) {
    if (!p) return fail(KYRO_EINVAL, "%s: params is null", call);
    if (p->block_size <= 0 || p->batch_size < 0 || p->num_state_rows <= 0 || p->max_state_blocks <= 0 ||
        p->num_blocks <= 0 || p->pool_capacity < 0 || (extend && (p->max_blocks_per_seq <= 0 || p->max_rows < 0)))
        return fail(KYRO_EINVAL, "%s: sizes must be positive (batch_size, pool_capacity, max_rows >= 0)", call);
    if (p->num_state_rows > kyro::kTablesMaxRows)
        return fail(KYRO_EUNSUPPORTED, "%s: num_state_rows %d (at most %d)", call, p->num_state_rows, kyro::kTablesMaxRows);
    if ((int64_t)p->max_state_blocks * p->block_size > INT32_MAX)
        return fail(KYRO_EUNSUPPORTED, "%s: a request of more than 2^31 tokens (max_state_blocks x block_size)", call);
    if (!state_rows && p->batch_size > p->num_state_rows)
        return fail(KYRO_EINVAL, "%s: without state_rows every entry of the batch needs a request of the state", call);
    a.B = p->batch_size;
    a.num_rows = p->num_state_rows;
    a.state_blocks = p->max_state_blocks;
    a.width = p->max_blocks_per_seq;
    a.bs = p->block_size;
    a.bs_shift = -1;
    for (int i = 0; i < 31; ++i)
        if (a.bs == 1 << i) a.bs_shift = i;
    a.num_blocks = p->num_blocks;
    a.pool_cap = p->pool_capacity;
    a.max_rows = p->max_rows;
    a.kept_plus = p->kept_plus;
    return KYRO_OK;
}

size_t tables_bytes(const kyro::TablesArgs& a) { return (size_t)a.B * sizeof(kyro::TablesEntry); }

// The state's arrays, which every call takes.
int bind_state(const char* call, const int32_t* state_rows, int32_t* requests, const int64_t* blocks, const int64_t* pool,
               int32_t* pool_count, bool extend, kyro::TablesArgs& a, Ranges& mem) {
    if (!requests || !blocks || !pool_count || (!pool && a.pool_cap > 0)) return fail(KYRO_EINVAL, "%s: null device pointer", call);
    if (reinterpret_cast<uintptr_t>(requests) % 16 != 0)
        return fail(KYRO_EINVAL, "%s: requests must be on a 16-byte boundary", call);
    a.state_rows = state_rows;
    a.requests = reinterpret_cast<int4*>(requests);
    a.blocks = const_cast<int64_t*>(blocks);
    a.pool = pool;
    a.pool_out = const_cast<int64_t*>(pool);
    a.pool_count = pool_count;
    mem.add("state_rows", state_rows, (uint64_t)a.B * 4, false);
    mem.add("requests", requests, (uint64_t)a.num_rows * 16, true);
    mem.add("blocks", blocks, (uint64_t)a.num_rows * a.state_blocks * 8, extend);
    mem.add("pool", pool, (uint64_t)a.pool_cap * 8, !extend);
    mem.add("pool_count", pool_count, 4, true);
    return KYRO_OK;
}

int too_large(const char* call) { return fail(KYRO_EUNSUPPORTED, "%s: the batch's tables are more than one launch carries", call); }

}  // namespace

extern "C" {

int kyro_tables_extend(kyro_ctx ctx, const kyro_tables_params* params, const int32_t* state_rows, const int32_t* new_rows,
                       int32_t* requests, int64_t* blocks, const int64_t* pool, int32_t* pool_count, int64_t* block_table,
                       int64_t* context_lens, int32_t* q_start_loc, int64_t* positions, int64_t* slots) {
    return guarded([&]() -> int {
        constexpr const char* call = "tables_extend";
        kyro::TablesArgs a{};
        if (int rc = tables_setup(params, call, true, state_rows, a)) return rc;
        if (a.B == 0) return check_ctx(ctx);
        Ranges mem;
        if (int rc = bind_state(call, state_rows, requests, blocks, pool, pool_count, true, a, mem)) return rc;
        if (!new_rows || !block_table || !context_lens || !q_start_loc) return fail(KYRO_EINVAL, "%s: null device pointer", call);
        a.new_rows = new_rows;
        a.table = block_table;
        a.ctx_lens = context_lens;
        a.q_start = q_start_loc;
        a.positions = positions;
        a.slots = slots;
        mem.add("new_rows", new_rows, (uint64_t)a.B * 4, false);
        mem.add("block_table", block_table, (uint64_t)a.B * a.width * 8, true);
        mem.add("context_lens", context_lens, (uint64_t)a.B * 8, true);
        mem.add("q_start_loc", q_start_loc, (uint64_t)(a.B + 1) * 4, true);
        mem.add("positions", positions, (uint64_t)a.max_rows * 8, true);
        mem.add("slots", slots, (uint64_t)a.max_rows * 8, true);
        if (int rc = mem.check(call)) return rc;
        int64_t table_wgs;
        if (kyro::tables_fill_wgs(a, table_wgs) > (int64_t)(0xffffffffu / 256)) return too_large(call);
        if (int rc = check_ctx(ctx)) return rc;  // last, so that a host without a device can have the rest checked
        DeviceGuard dg(ctx->device);
        KYRO_HIP(dg.status);
        if (int rc = ensure_arena(ctx, tables_bytes(a))) return rc;
        a.entries = static_cast<kyro::TablesEntry*>(ctx->arena);
        a.err = ctx->err;
        KYRO_HIP(kyro::launch_tables_extend(a, ctx->stream));
        return KYRO_OK;
    });
}

int kyro_tables_keep(kyro_ctx ctx, const kyro_tables_params* params, const int32_t* state_rows, const int64_t* context_lens,
                     const int32_t* q_start_loc, const int32_t* kept, int32_t* requests, const int64_t* blocks, int64_t* pool,
                     int32_t* pool_count, int64_t* out_context_lens) {
    return guarded([&]() -> int {
        constexpr const char* call = "tables_keep";
        kyro::TablesArgs a{};
        if (int rc = tables_setup(params, call, false, state_rows, a)) return rc;
        if (a.B == 0) return check_ctx(ctx);
        Ranges mem;
        if (int rc = bind_state(call, state_rows, requests, blocks, pool, pool_count, false, a, mem)) return rc;
        if (!context_lens || !q_start_loc || !kept || !out_context_lens) return fail(KYRO_EINVAL, "%s: null device pointer", call);
        a.ctx_lens = const_cast<int64_t*>(context_lens);
        a.q_start = const_cast<int32_t*>(q_start_loc);
        a.kept = kept;
        a.out_ctx = out_context_lens;
        if (out_context_lens != context_lens) mem.add("context_lens", context_lens, (uint64_t)a.B * 8, false);
        mem.add("q_start_loc", q_start_loc, (uint64_t)(a.B + 1) * 4, false);
        mem.add("kept", kept, (uint64_t)a.B * 4, false);
        mem.add("out_context_lens", out_context_lens, (uint64_t)a.B * 8, true);
        if (int rc = mem.check(call)) return rc;
        if (int rc = check_ctx(ctx)) return rc;
        DeviceGuard dg(ctx->device);
        KYRO_HIP(dg.status);
        a.err = ctx->err;
        KYRO_HIP(kyro::launch_tables_keep(a, ctx->stream));
        return KYRO_OK;
    });
}

int kyro_tables_release(kyro_ctx ctx, const kyro_tables_params* params, const int32_t* state_rows, int32_t* requests,
                        const int64_t* blocks, int64_t* pool, int32_t* pool_count) {
    return guarded([&]() -> int {
        constexpr const char* call = "tables_release";
        kyro::TablesArgs a{};
        if (int rc = tables_setup(params, call, false, state_rows, a)) return rc;
        if (a.B == 0) return check_ctx(ctx);
        Ranges mem;
        if (int rc = bind_state(call, state_rows, requests, blocks, pool, pool_count, false, a, mem)) return rc;
        if (int rc = mem.check(call)) return rc;
        if (kyro::tables_free_wgs(a) > (int64_t)(0xffffffffu / 256)) return too_large(call);
        if (int rc = check_ctx(ctx)) return rc;
        DeviceGuard dg(ctx->device);
        KYRO_HIP(dg.status);
        if (int rc = ensure_arena(ctx, tables_bytes(a))) return rc;
        a.entries = static_cast<kyro::TablesEntry*>(ctx->arena);
        a.err = ctx->err;
        KYRO_HIP(kyro::launch_tables_release(a, ctx->stream));
        return KYRO_OK;
    });
}

int kyro_tables_workspace(const kyro_tables_params* params, size_t* bytes) {
    return guarded([&]() -> int {
        if (!bytes) return fail(KYRO_EINVAL, "tables_workspace: bytes is null");
        *bytes = 0;
        kyro::TablesArgs a{};
        if (int rc = tables_setup(params, "tables_workspace", false, params, a)) return rc;
        *bytes = tables_bytes(a);
        return KYRO_OK;
    });
}

}  // extern "C"
