// C ABI of the block manager, the prefix cache, the device block-table writer and block copies
// (include/kyro_blocks.h), and of the accumulated attention weights and the eviction by them
// (include/kyro_evict.h), and of the block tables that live on the GPU (include/kyro_tables.h).
// Host logic lives in block_manager.cpp; this file validates arguments,
// converts statuses and queues the device work on the context's stream.
#include <algorithm>
#include <cmath>
#include <vector>

#include "block_manager.hpp"
#include "context.hpp"
#include "kernels.hpp"
#include "kyro_blocks.h"
#include "kyro_evict.h"
#include "kyro_tables.h"

using namespace kyro::rt;

struct kyro_bm_s {
    kyro::bm::BlockManager m;
    // Per block: (call number << 32) | (1 + the request that listed it last), for telling
    // kyro_bm_write_tables' callers whether two requests share a block.
    std::vector<uint64_t> seen;
    uint32_t calls = 0;
    kyro_bm_s(int bs, int64_t gpu, int64_t cpu) : m(bs, gpu, cpu), seen((size_t)gpu, 0) {}
};

struct kyro_radix_s {
    kyro::bm::RadixCache c;
    kyro_radix_s(int bs, int64_t cap) : c(bs, cap) {}
};

namespace {

int bm_status(int s, const char* what, uint64_t rid) {
    if (s == kyro::bm::OK) return KYRO_OK;
    if (s == kyro::bm::ENOSPACE)
        return fail(KYRO_ENOSPACE, "%s: not enough free KV blocks for request %llu", what, (unsigned long long)rid);
    return fail(KYRO_EINVAL, "%s: bad request %llu or size (unknown id, id in use, or out of range)", what,
                (unsigned long long)rid);
}

int copy_match(const std::pair<std::vector<int64_t>, int64_t>& m, int64_t* out, int64_t cap,
               int64_t* out_n, int64_t* out_matched) {
    const int64_t nb = (int64_t)m.first.size();
    if (out_n) *out_n = nb;
    if (out_matched) *out_matched = m.second;
    if (out) std::copy(m.first.begin(), m.first.begin() + std::min(nb, std::max<int64_t>(cap, 0)), out);
    return KYRO_OK;
}

uintptr_t at(const void* p) { return reinterpret_cast<uintptr_t>(p); }

// Do two arrays of `bytes` share memory without being the same one?
bool half_over(const void* x, const void* y, size_t bytes) {
    return x != y && at(x) < at(y) + bytes && at(y) < at(x) + bytes;
}

// Tokens a sequence may have: as many as its table and its state hold.
int64_t token_cap(int32_t max_blocks, int32_t block_size, int32_t max_tokens) {
    return std::min((int64_t)max_blocks * block_size, (int64_t)max_tokens);
}

// Sizes, variant and scratch of a kyro_attn_weights call, from its params alone.
int weights_setup(const kyro_attn_weights_params* p, bool has_q_start, int num_cus, kyro::AttnWeightsArgs& a,
                  size_t& bytes) {
    bytes = 0;
    if (!p) return fail(KYRO_EINVAL, "attn_weights: params is null");
    if (p->block_size <= 0 || p->num_heads <= 0 || p->head_dim <= 0 || p->num_kv_heads <= 0 || p->batch_size < 0 ||
        p->total_q < 0 || p->max_blocks_per_seq <= 0 || p->num_blocks <= 0 || p->max_q_len < 0 ||
        p->num_state_rows <= 0 || p->max_tokens <= 0)
        return fail(KYRO_EINVAL, "attn_weights: sizes must be positive (batch_size, total_q, max_q_len >= 0)");
    if (p->num_heads % p->num_kv_heads != 0)
        return fail(KYRO_EINVAL, "attn_weights: num_heads %d is not a multiple of num_kv_heads %d", p->num_heads,
                    p->num_kv_heads);
    if (p->head_dim % 8 != 0 || p->head_dim > 256)
        return fail(KYRO_EUNSUPPORTED, "attn_weights: head_dim %d is not supported (multiples of 8 up to 256)", p->head_dim);
    if (p->dtype != KYRO_F32 && p->dtype != KYRO_BF16) return fail(KYRO_EINVAL, "attn_weights: unknown dtype");
    if (!(p->scale >= 0.f) || !std::isfinite(p->scale))
        return fail(KYRO_EINVAL, "attn_weights: scale must be finite and >= 0");
    if (!has_q_start && p->total_q != p->batch_size)
        return fail(KYRO_EINVAL, "attn_weights: without q_start_loc total_q must equal batch_size");
    a.B = p->batch_size;
    a.H = p->num_heads;
    a.Hkv = p->num_kv_heads;
    a.group = a.H / a.Hkv;
    a.D = p->head_dim;
    a.bs = p->block_size;
    a.bs_shift = -1;
    for (int i = 0; i < 31; ++i)
        if (a.bs == 1 << i) a.bs_shift = i;
    a.max_blocks = p->max_blocks_per_seq;
    a.num_blocks = p->num_blocks;
    a.total_q = p->total_q;
    a.max_q_len = !has_q_start ? 1 : p->max_q_len > 0 ? p->max_q_len : p->total_q;
    a.num_state_rows = p->num_state_rows;
    a.max_tokens = p->max_tokens;
    a.causal = p->causal != 0;
    a.bf16 = p->dtype == KYRO_BF16;
    a.cap = token_cap(a.max_blocks, a.bs, a.max_tokens);
    const double scale = p->scale != 0.f ? (double)p->scale : 1.0 / std::sqrt((double)a.D);
    a.scale_log2 = (float)(scale * 1.4426950408889634);
    if (!std::isnormal(a.scale_log2))
        return fail(KYRO_EINVAL, "attn_weights: scale %g is too small or too large for 32 bits", (double)p->scale);
    if (a.B == 0 || a.total_q == 0) return KYRO_OK;
    const int64_t rows = (int64_t)std::min(a.max_q_len, a.total_q) * a.group;
    const double block_elems = (double)a.Hkv * a.bs * a.D;
    if (a.cap > (1 << 30) || rows > (1 << 30) || rows * a.group > INT32_MAX || (int64_t)a.total_q * a.H > INT32_MAX ||
        block_elems > UINT32_MAX)
        return fail(KYRO_EUNSUPPORTED, "attn_weights: more tokens or query rows than one launch carries");
    a.block_elems = (uint32_t)block_elems;
    a.group_magic = a.group > 1 ? (uint32_t)((((uint64_t)1 << 32) + a.group - 1) / a.group) : 0;
    const int most_few = kyro::attn_weights_few_rows(a.bf16, a.D), hold = kyro::attn_weights_many_hold(a.bf16, a.D);
    const bool many = rows > most_few;
    a.few_rows = rows <= 16 ? 16 : rows <= 32 ? 32 : most_few;
    const int64_t groups = many ? (rows + hold - 1) / hold : 1;
    const auto items = [&](int64_t chunk) { return a.B * ((a.cap + chunk - 1) / chunk) * a.Hkv * groups; };
    const auto part_bytes = [&](int64_t chunk) {
        return (size_t)((a.cap + chunk - 1) / chunk) * a.total_q * a.H * sizeof(float2);
    };
    a.kept_rows = (int)((rows + 3) / 4 * 4);
    // Scores are kept where writing and reading them (8 bytes a row and token) is enough less than reading the
    // keys again: 64 x 4096 tokens, 32/8 heads of 128 in bf16 (256 bytes a key) took 231 us kept and 205 us
    // computed again at 32 rows; f32 keys of 512 bytes 87 and 133 us at 5 rows.
    const bool keep = !many && (rows <= 16 || (rows <= 32 && 10 * a.kept_rows <= a.D * (a.bf16 ? 2 : 4)));
    // Chunks as long as they may be while there are a few for each CU: a chunk costs its start (a walk to its
    // sequence, its queries, its first keys), the last ones leave CUs idle. 8 x 2048 and 16 x 1024 tokens a CU
    // measured best on the two cases above.
    int64_t chunk = many && a.bf16 ? 128 : 64;
    while (chunk < (keep ? 1024 : 2048) && items(2 * chunk) >= (keep ? 8 : many ? 2 : 4) * num_cus) chunk *= 2;
    while (part_bytes(chunk) > ((size_t)64 << 20) && chunk < a.cap) chunk *= 2;
    a.chunk = (int)chunk;
    // 64 sequences' items are counted in 32 bits.
    if ((double)((a.cap + 63) / 64) * a.Hkv * groups * 64 > INT32_MAX)
        return fail(KYRO_EUNSUPPORTED, "attn_weights: more work items than one launch carries");
    // Where some sequences have fewer rows than the largest, the few-row kernels take those they can.
    const int64_t most = 8 * (int64_t)num_cus;
    const bool mixed = many && (int64_t)a.total_q < (int64_t)a.B * a.max_q_len;
    if (many && !mixed) a.few_rows = 0;
    a.few_items_most = many && !mixed ? 0 : a.B * ((a.cap + chunk - 1) / chunk) * a.Hkv;
    a.few_grid = (int)std::min(most, a.few_items_most);
    a.many_stat_grid = many ? (int)std::min(most, items(chunk)) : 0;
    // Few runs of tokens for the CUs (short contexts of many rows): the rows are split, into parts of at least
    // 128 (f32 products take eight times as long: 64), until there are two workgroups a CU.
    const int64_t runs = a.B * ((a.cap + hold - 1) / hold) * a.Hkv;
    a.row_parts = many ? (int)std::max<int64_t>(1, std::min<int64_t>((2 * num_cus + runs - 1) / runs, rows / (a.bf16 ? 128 : 64))) : 1;
    a.run_tokens = (a.cap + hold - 1) / hold * hold;
    a.many_sum_grid = many ? (int)std::min(most, runs * a.row_parts) : 0;
    bytes = align_up(part_bytes(chunk), 256) + (many ? align_up((size_t)a.total_q * a.H * sizeof(float), 256) : 0);
    if (a.row_parts > 1) bytes += align_up((size_t)a.row_parts * a.B * a.Hkv * a.run_tokens * sizeof(float), 256);
    if (keep) {  // at most 256 MiB of them: items past that are computed again
        const size_t item = (size_t)chunk * a.kept_rows * sizeof(float);
        a.kept_items = std::min<int64_t>(a.few_items_most, (int64_t)(((size_t)256 << 20) / item));
        bytes += align_up((size_t)a.kept_items * item, 256);
    }
    return KYRO_OK;
}

int evict_setup(const kyro_kv_evict_params* p, kyro::EvictArgs& a, size_t& bytes) {
    bytes = 0;
    if (!p) return fail(KYRO_EINVAL, "kv_evict: params is null");
    if (p->block_size <= 0 || p->num_kv_heads <= 0 || p->head_dim <= 0 || p->batch_size < 0 ||
        p->max_blocks_per_seq <= 0 || p->num_blocks <= 0 || p->num_state_rows <= 0 || p->max_tokens <= 0)
        return fail(KYRO_EINVAL, "kv_evict: sizes must be positive (batch_size >= 0)");
    if (p->head_dim % 8 != 0 || p->head_dim > 256)
        return fail(KYRO_EUNSUPPORTED, "kv_evict: head_dim %d is not supported (multiples of 8 up to 256)", p->head_dim);
    if (p->dtype != KYRO_F32 && p->dtype != KYRO_BF16) return fail(KYRO_EINVAL, "kv_evict: unknown dtype");
    if (p->budget <= 0 || p->sink < 0 || p->recent < 0 || (int64_t)p->sink + p->recent > p->budget)
        return fail(KYRO_EINVAL, "kv_evict: need budget > 0, sink >= 0, recent >= 0 and sink + recent <= budget");
    a.cap = token_cap(p->max_blocks_per_seq, p->block_size, p->max_tokens);
    // A grid has fewer than 2^32 threads, and a (sequence, kv head) a workgroup of 1024.
    if (a.cap > (1 << 30) || (int64_t)p->batch_size * p->num_kv_heads >= (1 << 22))
        return fail(KYRO_EUNSUPPORTED, "kv_evict: more tokens or sequences than one launch carries");
    a.B = p->batch_size;
    a.Hkv = p->num_kv_heads;
    a.bs = p->block_size;
    a.max_blocks = p->max_blocks_per_seq;
    a.num_blocks = p->num_blocks;
    a.num_state_rows = p->num_state_rows;
    a.max_tokens = p->max_tokens;
    a.row_vecs = p->head_dim * (p->dtype == KYRO_BF16 ? 2 : 4) / 16;
    a.budget = p->budget;
    a.sink = p->sink;
    a.recent = p->recent;
    a.max_moves = (int)std::max<int64_t>(0, std::min<int64_t>(a.budget, a.cap - a.budget));
    // A selecting workgroup copies what it moves (64 sequences of 8 heads, 256 moves of 512 bytes: 43 us; 16 + 32 in
    // two kernels), except where few of them would copy much each (64 of them, 900 moves: 42 us, 21 + 11 in two):
    // then about 4096 workgroups share the moves, each with at least 1024 vectors where the most tokens move.
    const int64_t units = std::max<int64_t>(1, (int64_t)a.B * a.Hkv);
    const bool own = units >= 128 || (int64_t)a.max_moves * a.row_vecs <= 8192;
    a.own_moves = own ? kyro::kEvictOwnMoves : 0;
    const int64_t left = std::max<int64_t>(0, (int64_t)a.max_moves - a.own_moves) * a.row_vecs;
    a.move_wgs = (int)std::max<int64_t>(1, std::min<int64_t>((4096 + units - 1) / units, (left + 1023) / 1024));
    bytes = align_up((size_t)a.B * a.Hkv * sizeof(int), 256) +
            align_up((size_t)a.B * a.Hkv * 2 * a.max_moves * sizeof(int32_t), 256);
    return KYRO_OK;
}

}  // namespace

extern "C" {

// ------------------------------------------------------------------------- prefix cache

int kyro_radix_create(int32_t block_size, int64_t max_capacity, kyro_radix* out) {
    return guarded([&]() -> int {
        if (!out) return fail(KYRO_EINVAL, "radix_create: out is null");
        *out = nullptr;
        if (block_size <= 0 || max_capacity < 0)
            return fail(KYRO_EINVAL, "radix_create: block_size must be > 0 and max_capacity >= 0");
        *out = new kyro_radix_s(block_size, max_capacity);
        return KYRO_OK;
    });
}

int kyro_radix_destroy(kyro_radix r) {
    return guarded([&]() -> int {
        delete r;
        return KYRO_OK;
    });
}

int kyro_radix_match_prefix(kyro_radix r, const uint32_t* tokens, int64_t n, int64_t* out_blocks,
                            int64_t cap, int64_t* out_num_blocks, int64_t* out_matched) {
    return guarded([&]() -> int {
        if (!r || n < 0 || (n > 0 && !tokens)) return fail(KYRO_EINVAL, "radix_match_prefix: bad arguments");
        return copy_match(r->c.match_prefix(tokens, n), out_blocks, cap, out_num_blocks, out_matched);
    });
}

int kyro_radix_insert(kyro_radix r, const uint32_t* tokens, int64_t n, const int64_t* blocks,
                      uint8_t* out_taken) {
    return guarded([&]() -> int {
        if (!r || n < 0 || (n > 0 && (!tokens || !blocks))) return fail(KYRO_EINVAL, "radix_insert: bad arguments");
        const std::vector<bool> taken = r->c.insert(tokens, n, blocks, nullptr);
        if (out_taken)
            for (size_t i = 0; i < taken.size(); ++i) out_taken[i] = taken[i] ? 1 : 0;
        return KYRO_OK;
    });
}

int kyro_radix_evict_lru(kyro_radix r, int64_t* out, int64_t cap, int64_t* out_n) {
    return guarded([&]() -> int {
        if (!r) return fail(KYRO_EINVAL, "radix_evict_lru: null handle");
        const std::vector<int64_t> ev = r->c.evict_lru();
        if (out_n) *out_n = (int64_t)ev.size();
        if (out) std::copy(ev.begin(), ev.begin() + std::min<int64_t>((int64_t)ev.size(), std::max<int64_t>(cap, 0)), out);
        return KYRO_OK;
    });
}

int64_t kyro_radix_num_cached_blocks(kyro_radix r) { return r ? r->c.num_cached_blocks() : -1; }

// ------------------------------------------------------------------------ block manager

int kyro_bm_create(int32_t block_size, int64_t num_gpu_blocks, int64_t num_cpu_blocks, kyro_bm* out) {
    return guarded([&]() -> int {
        if (!out) return fail(KYRO_EINVAL, "bm_create: out is null");
        *out = nullptr;
        if (block_size <= 0 || num_gpu_blocks < 0 || num_cpu_blocks < 0)
            return fail(KYRO_EINVAL, "bm_create: block_size must be > 0 and block counts >= 0");
        *out = new kyro_bm_s(block_size, num_gpu_blocks, num_cpu_blocks);
        return KYRO_OK;
    });
}

int kyro_bm_destroy(kyro_bm bm) {
    return guarded([&]() -> int {
        delete bm;
        return KYRO_OK;
    });
}

int kyro_bm_allocate_with_prefix(kyro_bm bm, uint64_t request_id, const uint32_t* tokens, int64_t n,
                                 int64_t* out_cached_tokens) {
    return guarded([&]() -> int {
        if (!bm || n < 0 || (n > 0 && !tokens) || !out_cached_tokens)
            return fail(KYRO_EINVAL, "bm_allocate_with_prefix: bad arguments");
        return bm_status(bm->m.allocate_with_prefix(request_id, tokens, n, out_cached_tokens),
                         "bm_allocate_with_prefix", request_id);
    });
}

int kyro_bm_allocate(kyro_bm bm, uint64_t request_id, int64_t num_tokens) {
    return guarded([&]() -> int {
        if (!bm) return fail(KYRO_EINVAL, "bm_allocate: null handle");
        return bm_status(bm->m.allocate(request_id, num_tokens), "bm_allocate", request_id);
    });
}

int kyro_bm_append_slots(kyro_bm bm, uint64_t request_id, int64_t n) {
    return guarded([&]() -> int {
        if (!bm) return fail(KYRO_EINVAL, "bm_append_slots: null handle");
        return bm_status(bm->m.append_slots(request_id, n), "bm_append_slots", request_id);
    });
}

int kyro_bm_truncate(kyro_bm bm, uint64_t request_id, int64_t num_tokens) {
    return guarded([&]() -> int {
        if (!bm) return fail(KYRO_EINVAL, "bm_truncate: null handle");
        return bm_status(bm->m.truncate(request_id, num_tokens), "bm_truncate", request_id);
    });
}

int kyro_bm_make_private(kyro_bm bm, uint64_t request_id) {
    return guarded([&]() -> int {
        if (!bm) return fail(KYRO_EINVAL, "bm_make_private: null handle");
        return bm_status(bm->m.make_private(request_id, INT64_MAX), "bm_make_private", request_id);
    });
}

int kyro_bm_make_private_front(kyro_bm bm, uint64_t request_id, int64_t num_tokens) {
    return guarded([&]() -> int {
        if (!bm) return fail(KYRO_EINVAL, "bm_make_private_front: null handle");
        return bm_status(bm->m.make_private(request_id, num_tokens), "bm_make_private_front", request_id);
    });
}

int kyro_bm_free(kyro_bm bm, uint64_t request_id, int32_t cache_prompt) {
    return guarded([&]() -> int {
        if (!bm) return fail(KYRO_EINVAL, "bm_free: null handle");
        return bm_status(bm->m.free(request_id, cache_prompt != 0), "bm_free", request_id);
    });
}

int kyro_bm_request_blocks(kyro_bm bm, uint64_t request_id, int64_t* out, int64_t cap, int64_t* out_n,
                           int64_t* out_num_tokens) {
    return guarded([&]() -> int {
        if (!bm) return fail(KYRO_EINVAL, "bm_request_blocks: null handle");
        const kyro::bm::Request* r = bm->m.find(request_id);
        if (!r) return fail(KYRO_EINVAL, "bm_request_blocks: unknown request %llu", (unsigned long long)request_id);
        const int64_t nb = (int64_t)r->blocks.size();
        if (out_n) *out_n = nb;
        if (out_num_tokens) *out_num_tokens = r->num_tokens;
        if (out) std::copy(r->blocks.begin(), r->blocks.begin() + std::min(nb, std::max<int64_t>(cap, 0)), out);
        return KYRO_OK;
    });
}

int kyro_bm_take_copies(kyro_bm bm, int64_t* src, int64_t* dst, int64_t cap, int64_t* out_n) {
    return guarded([&]() -> int {
        if (!bm || !out_n) return fail(KYRO_EINVAL, "bm_take_copies: bad arguments");
        // Peek first: nothing is taken unless it all fits.
        std::vector<std::pair<int64_t, int64_t>> c = bm->m.take_copies_peek();
        *out_n = (int64_t)c.size();
        if ((int64_t)c.size() > cap || (!c.empty() && (!src || !dst))) return KYRO_OK;
        c = bm->m.take_copies();
        for (size_t i = 0; i < c.size(); ++i) {
            src[i] = c[i].first;
            dst[i] = c[i].second;
        }
        return KYRO_OK;
    });
}

int64_t kyro_bm_num_free_blocks(kyro_bm bm) { return bm ? bm->m.num_free_blocks() : -1; }

int kyro_bm_check(kyro_bm bm) {
    return guarded([&]() -> int {
        if (!bm) return fail(KYRO_EINVAL, "bm_check: null handle");
        const std::string e = bm->m.check();
        if (!e.empty()) return fail(KYRO_EINVAL, "bm_check: %s", e.c_str());
        return KYRO_OK;
    });
}

int64_t kyro_bm_num_cached_blocks(kyro_bm bm) { return bm ? bm->m.cache().num_cached_blocks() : -1; }

int kyro_bm_match_prefix(kyro_bm bm, const uint32_t* tokens, int64_t n, int64_t* out_blocks, int64_t cap,
                         int64_t* out_num_blocks, int64_t* out_matched) {
    return guarded([&]() -> int {
        if (!bm || n < 0 || (n > 0 && !tokens)) return fail(KYRO_EINVAL, "bm_match_prefix: bad arguments");
        return copy_match(bm->m.cache().match_prefix(tokens, n), out_blocks, cap, out_num_blocks, out_matched);
    });
}

int kyro_bm_write_tables(kyro_bm bm, kyro_ctx ctx, const uint64_t* request_ids, int32_t B, int32_t max_blocks,
                         int64_t* block_table, int64_t* context_lens, int32_t* out_shared) {
    return guarded([&]() -> int {
        if (int rc = check_ctx(ctx)) return rc;
        if (!bm || B < 0 || max_blocks <= 0 || (B > 0 && (!request_ids || !block_table)))
            return fail(KYRO_EINVAL, "bm_write_tables: bad arguments");
        if (out_shared) *out_shared = 0;
        if (B == 0) return KYRO_OK;
        if (++bm->calls == 0) {  // the call counter wrapped: forget every older mark
            std::fill(bm->seen.begin(), bm->seen.end(), 0);
            bm->calls = 1;
        }
        const uint64_t call = (uint64_t)bm->calls << 32;
        int32_t shared = 0;
        std::vector<int64_t> table((size_t)B * max_blocks, 0), lens((size_t)B, 0);
        for (int32_t b = 0; b < B; ++b) {
            const kyro::bm::Request* r = bm->m.find(request_ids[b]);
            if (!r)
                return fail(KYRO_EINVAL, "bm_write_tables: unknown request %llu", (unsigned long long)request_ids[b]);
            if ((int64_t)r->blocks.size() > max_blocks)
                return fail(KYRO_EINVAL, "bm_write_tables: request %llu holds %zu blocks > max_blocks %d",
                            (unsigned long long)request_ids[b], r->blocks.size(), max_blocks);
            std::copy(r->blocks.begin(), r->blocks.end(), table.begin() + (size_t)b * max_blocks);
            lens[(size_t)b] = r->num_tokens;
            for (const int64_t blk : r->blocks) {
                if (blk < 0 || (size_t)blk >= bm->seen.size()) continue;
                uint64_t& s = bm->seen[(size_t)blk];
                const uint64_t mine = call | (uint64_t)(b + 1);
                if ((s & ~0xffffffffull) == call && s != mine) shared = 1;
                s = mine;
            }
        }
        if (out_shared) *out_shared = shared;
        DeviceGuard dg(ctx->device);
        KYRO_HIP(dg.status);
        Upload ups[2] = {{block_table, table.data(), table.size() * sizeof(int64_t)},
                         {context_lens, lens.data(), context_lens ? lens.size() * sizeof(int64_t) : 0}};
        return stage_uploads(ctx, ups, context_lens ? 2 : 1);
    });
}

int kyro_bm_prefix_groups(kyro_bm bm, const uint64_t* request_ids, int32_t B, int32_t* order, int32_t* group_starts,
                          int32_t* group_blocks, int32_t* num_groups) {
    return guarded([&]() -> int {
        if (!bm || B < 0 || !group_starts || !num_groups || (B > 0 && (!request_ids || !order || !group_blocks)))
            return fail(KYRO_EINVAL, "bm_prefix_groups: bad arguments");
        std::vector<const std::vector<int64_t>*> lists((size_t)B);
        for (int32_t b = 0; b < B; ++b) {
            const kyro::bm::Request* r = bm->m.find(request_ids[b]);
            if (!r)
                return fail(KYRO_EINVAL, "bm_prefix_groups: unknown request %llu", (unsigned long long)request_ids[b]);
            lists[(size_t)b] = &r->blocks;
        }
        const std::vector<kyro::bm::PrefixGroup> groups = kyro::bm::prefix_groups(lists);
        int32_t at = 0;
        for (size_t g = 0; g < groups.size(); ++g) {
            group_starts[g] = at;
            group_blocks[g] = (int32_t)groups[g].blocks;
            for (const int32_t b : groups[g].members) order[at++] = b;
        }
        group_starts[groups.size()] = at;
        *num_groups = (int32_t)groups.size();
        return KYRO_OK;
    });
}

// ------------------------------------------------------------------------------- copies

int kyro_copy_blocks(kyro_ctx ctx, const kyro_copy_blocks_params* p, void* key_cache, void* value_cache,
                     const int64_t* src, const int64_t* dst, int64_t n) {
    return guarded([&]() -> int {
        if (int rc = check_ctx(ctx)) return rc;
        if (!p || n < 0) return fail(KYRO_EINVAL, "copy_blocks: bad arguments");
        if (n == 0) return KYRO_OK;
        if (!src || !dst || !key_cache || !value_cache) return fail(KYRO_EINVAL, "copy_blocks: null pointer");
        if (p->block_size <= 0 || p->num_kv_heads <= 0 || p->head_dim <= 0 || p->num_blocks <= 0 ||
            (p->dtype != KYRO_F32 && p->dtype != KYRO_BF16))
            return fail(KYRO_EINVAL, "copy_blocks: bad params");
        const size_t elem = p->dtype == KYRO_F32 ? 4 : 2;
        const size_t slab = (size_t)p->num_kv_heads * p->block_size * p->head_dim * elem;
        if (slab % 16 != 0) return fail(KYRO_EUNSUPPORTED, "copy_blocks: a block is not a multiple of 16 bytes");
        if ((reinterpret_cast<uintptr_t>(key_cache) | reinterpret_cast<uintptr_t>(value_cache)) % 16 != 0)
            return fail(KYRO_EINVAL, "copy_blocks: caches must be 16-byte aligned");
        std::vector<int64_t> pairs((size_t)(2 * n));
        std::vector<char> is_src((size_t)p->num_blocks, 0);
        for (int64_t i = 0; i < n; ++i) {
            if (src[i] < 0 || src[i] >= p->num_blocks || dst[i] < 0 || dst[i] >= p->num_blocks)
                return fail(KYRO_EINVAL, "copy_blocks: block id outside [0, %d)", p->num_blocks);
            pairs[(size_t)i] = src[i];
            pairs[(size_t)(n + i)] = dst[i];
            is_src[(size_t)src[i]] = 1;
        }
        for (int64_t i = 0; i < n; ++i)
            if (is_src[(size_t)dst[i]]) return fail(KYRO_EINVAL, "copy_blocks: block %lld is both a source and a destination",
                                                    (long long)dst[i]);
        DeviceGuard dg(ctx->device);
        KYRO_HIP(dg.status);
        kyro::CopyBlocksArgs a{};
        if (n <= kyro::kCopyInline) {  // the pairs travel in the kernel arguments: no upload
            a.pairs = nullptr;
            for (int64_t i = 0; i < n; ++i) {
                a.inl[0][i] = (int32_t)src[i];
                a.inl[1][i] = (int32_t)dst[i];
            }
        } else {
            const size_t pair_bytes = pairs.size() * sizeof(int64_t);
            if (int rc = ensure_arena(ctx, pair_bytes)) return rc;
            Upload up = {ctx->arena, pairs.data(), pair_bytes};
            if (int rc = stage_uploads(ctx, &up, 1)) return rc;
            a.pairs = static_cast<const int64_t*>(ctx->arena);
        }
        a.n = n;
        a.slab_vecs = (int64_t)(slab / 16);
        a.kc = static_cast<uint4*>(key_cache);
        a.vc = static_cast<uint4*>(value_cache);
        KYRO_HIP(kyro::launch_copy_blocks(a, ctx->stream));
        return KYRO_OK;
    });
}

// ----------------------------------------------------- attention weights and eviction

int kyro_attn_weights(kyro_ctx ctx, const kyro_attn_weights_params* p, const void* query, const int32_t* q_start_loc,
                      const int64_t* row_positions, const void* key_cache, const int64_t* block_table,
                      const int64_t* context_lens, const int32_t* state_rows, const float* weights,
                      float* out_weights, int32_t* positions) {
    return guarded([&]() -> int {
        kyro::AttnWeightsArgs a{};
        size_t bytes = 0;
        if (int rc = weights_setup(p, q_start_loc != nullptr, ctx ? ctx->num_cus : 256, a, bytes)) return rc;
        // Without rows nothing is gained; weights that go elsewhere are taken along.
        if (a.B == 0 || (a.total_q == 0 && weights == out_weights)) return check_ctx(ctx);
        if ((!query && a.total_q) || !key_cache || !block_table || !context_lens || !weights || !out_weights || !positions)
            return fail(KYRO_EINVAL, "attn_weights: null device pointer");
        if ((at(query) | at(key_cache)) % 16 != 0)
            return fail(KYRO_EINVAL, "attn_weights: query and key_cache must be 16-byte aligned");
        if (!state_rows && a.B > a.num_state_rows)
            return fail(KYRO_EINVAL, "attn_weights: without state_rows the batch needs a state row each");
        if (half_over(weights, out_weights, (size_t)a.num_state_rows * a.Hkv * a.max_tokens * sizeof(float)))
            return fail(KYRO_EINVAL, "attn_weights: out_weights overlaps weights (only weights itself may)");
        if (int rc = check_ctx(ctx)) return rc;  // last, so that a host without a device can have the rest checked
        a.q = query;
        a.q_start = q_start_loc;
        a.row_pos = row_positions;
        a.k = key_cache;
        a.table = block_table;
        a.ctx_lens = context_lens;
        a.state_rows = state_rows;
        a.w = weights;
        a.out_w = out_weights;
        a.positions = positions;
        DeviceGuard dg(ctx->device);
        KYRO_HIP(dg.status);
        if (int rc = ensure_arena(ctx, bytes)) return rc;
        if (a.total_q > 0) {
            char* base = static_cast<char*>(ctx->arena);
            a.part = reinterpret_cast<float2*>(base);
            base += align_up((size_t)((a.cap + a.chunk - 1) / a.chunk) * a.total_q * a.H * sizeof(float2), 256);
            if (a.many_stat_grid) {
                a.lse = reinterpret_cast<float*>(base);
                base += align_up((size_t)a.total_q * a.H * sizeof(float), 256);
            }
            // A call has either parts of sums or kept scores.
            a.row_sums = a.kept = reinterpret_cast<float*>(base);
        }
        if (weights != out_weights && q_start_loc)
            a.idle = a.many_stat_grid || a.total_q == 0 ? kyro::kIdleMerge
                     : a.kept_items                     ? kyro::kIdleKeptSum
                                                        : kyro::kIdleFewSum;
        a.err = ctx->err;
        KYRO_HIP(kyro::launch_attn_weights(a, ctx->stream));
        return KYRO_OK;
    });
}

int kyro_attn_weights_workspace(kyro_ctx ctx, const kyro_attn_weights_params* p, int has_q_start_loc, size_t* bytes) {
    return guarded([&]() -> int {
        if (!bytes) return fail(KYRO_EINVAL, "attn_weights_workspace: bytes is null");
        kyro::AttnWeightsArgs a{};
        return weights_setup(p, has_q_start_loc != 0, ctx ? ctx->num_cus : 256, a, *bytes);
    });
}

int kyro_kv_evict(kyro_ctx ctx, const kyro_kv_evict_params* p, void* key_cache, void* value_cache,
                  const int64_t* block_table, const int64_t* context_lens, const int32_t* state_rows,
                  const float* weights, const int32_t* positions, float* out_weights, int32_t* out_positions,
                  int64_t* out_context_lens) {
    return guarded([&]() -> int {
        kyro::EvictArgs a{};
        size_t bytes = 0;
        if (int rc = evict_setup(p, a, bytes)) return rc;
        if (a.B == 0) return check_ctx(ctx);
        if (!key_cache || !value_cache || !block_table || !context_lens || !weights || !positions || !out_weights ||
            !out_positions || !out_context_lens)
            return fail(KYRO_EINVAL, "kv_evict: null device pointer");
        if ((at(key_cache) | at(value_cache)) % 16 != 0) return fail(KYRO_EINVAL, "kv_evict: caches must be 16-byte aligned");
        if (!state_rows && a.B > a.num_state_rows)
            return fail(KYRO_EINVAL, "kv_evict: without state_rows the batch needs a state row each");
        const size_t state = (size_t)a.num_state_rows * a.Hkv * a.max_tokens * 4;
        if (half_over(weights, out_weights, state) || half_over(positions, out_positions, state) ||
            at(weights) == at(out_positions) || at(positions) == at(out_weights) || at(out_weights) == at(out_positions) ||
            half_over(weights, out_positions, state) || half_over(positions, out_weights, state) ||
            half_over(out_weights, out_positions, state))
            return fail(KYRO_EINVAL, "kv_evict: out_weights and out_positions overlap an input (only their own input may)");
        const size_t lens = (size_t)a.B * sizeof(int64_t);
        if (context_lens == out_context_lens || half_over(context_lens, out_context_lens, lens))
            return fail(KYRO_EINVAL, "kv_evict: out_context_lens overlaps context_lens");
        if (int rc = check_ctx(ctx)) return rc;  // last, so that a host without a device can have the rest checked
        a.kc = static_cast<uint4*>(key_cache);
        a.vc = static_cast<uint4*>(value_cache);
        a.table = block_table;
        a.ctx_lens = context_lens;
        a.state_rows = state_rows;
        a.weights = weights;
        a.positions = positions;
        a.out_weights = out_weights;
        a.out_positions = out_positions;
        a.out_ctx_lens = out_context_lens;
        DeviceGuard dg(ctx->device);
        KYRO_HIP(dg.status);
        if (int rc = ensure_arena(ctx, bytes)) return rc;
        a.num_moves = static_cast<int*>(ctx->arena);
        a.moves = reinterpret_cast<int32_t*>(static_cast<char*>(ctx->arena) +
                                             align_up((size_t)a.B * a.Hkv * sizeof(int), 256));
        a.err = ctx->err;
        KYRO_HIP(kyro::launch_kv_evict(a, ctx->stream));
        return KYRO_OK;
    });
}

int kyro_kv_evict_workspace(const kyro_kv_evict_params* p, size_t* bytes) {
    return guarded([&]() -> int {
        if (!bytes) return fail(KYRO_EINVAL, "kv_evict_workspace: bytes is null");
        kyro::EvictArgs a{};
        return evict_setup(p, a, *bytes);
    });
}

}  // extern "C"

// ------------------------------------------------------------------------------- tables on the GPU (kyro_tables.h)

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
    if (p->max_state_blocks > kyro::kTablesMaxWidth || (extend && p->max_blocks_per_seq > kyro::kTablesMaxWidth))
        return fail(KYRO_EUNSUPPORTED, "%s: rows of at most %d blocks", call, kyro::kTablesMaxWidth);
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
        if (a.B > (int)(0xffffffffu / 256)) return too_large(call);  // as for the others, with a workgroup an entry
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
