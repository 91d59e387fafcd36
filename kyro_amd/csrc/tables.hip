// Block tables, row ranges and cache slots of a step from the requests' own records, and the pool of free
// blocks (include/kyro_tables.h).
//
// Everything that depends on the order of the batch (rows before an entry, blocks taken or given back before it)
// is a prefix sum over the batch, so one workgroup works the batch out, 1024 entries at a time: it reads each
// entry's state row and record, checks them, scans rows and blocks, and updates records and pool count. What is
// left has no order: table rows, positions and slots are written by as many workgroups as they fill
// (tables_fill_kernel), or, where they are few, by the first one right away, which saves the second launch.
#include "common.hpp"

namespace kyro {

namespace {

constexpr int kTabThreads = 1024;
constexpr int kTabWaves = kTabThreads / 64;
constexpr int kFillThreads = 256;
constexpr int kFillEntries = 2048;  // table entries, rows or freed blocks of one fill workgroup

// What the scan hands to the fill, for each entry of the batch.
struct Entry {
    int row, held, total, base;  // request (-1: left out); blocks before and after; pool entry of the first
                                 // block taken (going down) or given back (going up)
    int q0, rows, ctx, tokens;   // its rows, context length with them, tokens before them
};
static_assert(sizeof(Entry) == kTablesEntryBytes, "scratch of an entry");

// Inclusive sum over the workgroup's threads, and the total. `part` holds kTabWaves values.
__device__ __forceinline__ int64_t block_scan(int64_t x, int64_t* part, int64_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    __syncthreads();  // everyone has left the last scan's part
    if (lane == 63) part[wave] = x;
    __syncthreads();
    int64_t before = 0;
    total = 0;
    for (int w = 0; w < kTabWaves; ++w) {
        before += w < wave ? part[w] : 0;
        total += part[w];
    }
    return before + x;
}

// The batch's state rows, checked: marks in LDS which requests are named, and which twice.
struct Names {
    uint32_t* once;   // bits of requests named
    uint32_t* twice;  // named again

    __device__ void mark(const TablesArgs& a, uint32_t* lds) {
        const int words = (a.num_rows + 31) / 32;
        once = lds;
        twice = lds + words;
        for (int i = threadIdx.x; i < 2 * words; i += kTabThreads) lds[i] = 0;
        __syncthreads();
        for (int b = threadIdx.x; b < a.B; b += kTabThreads) {
            const int r = a.state_rows ? a.state_rows[b] : b;
            if (r < 0 || r >= a.num_rows) continue;
            const uint32_t bit = 1u << (r & 31);
            if (atomicOr(&once[r >> 5], bit) & bit) atomicOr(&twice[r >> 5], bit);
        }
        __syncthreads();
    }

    // Request of entry b, or -1 for padding and for one that is not (latched).
    __device__ int request(const TablesArgs& a, int b) const {
        const int r = a.state_rows ? a.state_rows[b] : b;
        if (r < 0) return -1;
        if (r >= a.num_rows || ((twice[r >> 5] >> (r & 31)) & 1u)) {
            latch_error(a.err, ERR_STATE_ROW);
            return -1;
        }
        return r;
    }
};

// A request's record {tokens, held, shared, -}; false (latched) where the numbers do not fit each other.
__device__ __forceinline__ bool load_record(const TablesArgs& a, int r, int4& rec) {
    rec = a.requests[r];
    const bool ok = rec.x >= 0 && rec.z >= 0 && rec.z <= rec.y && rec.y <= a.state_blocks &&
                    (int64_t)rec.x <= (int64_t)rec.y * a.bs;
    if (!ok) latch_error(a.err, ERR_REQUEST);
    return ok;
}

__device__ __forceinline__ int pool_count(const TablesArgs& a) {
    const int n = *a.pool_count;
    if (n >= 0 && n <= a.pool_cap) return n;
    if (threadIdx.x == 0) latch_error(a.err, ERR_POOL);
    return -1;
}

// Entry i of a table row of entry e; a block that is new is the request's from now on.
__device__ __forceinline__ void fill_block(const TablesArgs& a, const Entry& e, int b, int i) {
    int64_t id = 0;
    if (e.row >= 0 && i < e.total) {
        int64_t* own = a.blocks + (size_t)e.row * a.state_blocks + i;
        if (i < e.held) {
            id = *own;
        } else {
            id = a.pool[e.base - (i - e.held)];
            *own = id;
        }
        if (id < 0 || id >= a.num_blocks) latch_error(a.err, ERR_BLOCK_ID);
    }
    a.table[(size_t)b * a.width + i] = id;
}

// Position and slot of row j of entry e.
__device__ __forceinline__ void fill_row(const TablesArgs& a, const Entry& e, int64_t i, int j) {
    int64_t position = -1, slot = -1;
    if (e.row >= 0 && j >= 0) {
        const int p = e.tokens + j;
        const int blk = a.bs_shift >= 0 ? p >> a.bs_shift : p / a.bs;
        const int64_t id = blk < e.held ? a.blocks[(size_t)e.row * a.state_blocks + blk] : a.pool[e.base - (blk - e.held)];
        position = p;
        slot = id * a.bs + (p - blk * a.bs);
    }
    if (a.positions) a.positions[i] = position;
    if (a.slots) a.slots[i] = slot;
}

// The entry that row i belongs to (the last one that starts at or before it), or -1 behind the last row.
template <typename Start>
__device__ __forceinline__ int entry_of_row(int B, int64_t i, Start&& start) {
    if (i >= start(B)) return -1;
    int lo = 0, hi = B - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (start(mid) <= i) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// ONE: the whole call (at most kTabThreads entries).
template <bool ONE>
__global__ __launch_bounds__(kTabThreads) void tables_extend_kernel(TablesArgs a) {
    extern __shared__ uint32_t names_lds[];
    __shared__ int64_t part[kTabWaves];
    __shared__ Entry held[ONE ? kTabThreads : 1];
    Names names;
    names.mark(a, names_lds);
    const int count = pool_count(a);
    int64_t rows_before = 0, need_before = 0;
    int64_t taken = 0;  // by the entries served
    for (int b0 = 0; b0 < a.B; b0 += kTabThreads) {
        const int b = b0 + threadIdx.x;
        const bool in = b < a.B;
        int r = -1, m = 0;
        int4 rec = make_int4(0, 0, 0, 0);
        if (in) {
            r = names.request(a, b);
            m = a.new_rows[b];
            if (m < 0) {
                latch_error(a.err, ERR_Q_LAYOUT);
                m = 0;
                r = -1;
            }
            if (r >= 0 && !load_record(a, r, rec)) r = -1;
        }
        int64_t rows_all, need_all;
        const int64_t rows_to = rows_before + block_scan(m, part, rows_all);
        const int64_t ctx = (int64_t)rec.x + m;
        if (r >= 0 && rows_to > a.max_rows) {
            latch_error(a.err, ERR_Q_LAYOUT);
            r = -1;
        }
        if (r >= 0 && ctx > (int64_t)min(a.width, a.state_blocks) * a.bs) {
            latch_error(a.err, ERR_CTX_LEN);
            r = -1;
        }
        const int64_t need = r >= 0 ? max((ctx + a.bs - 1) / a.bs - rec.y, (int64_t)0) : 0;
        const int64_t need_to = need_before + block_scan(need, part, need_all);
        bool served = r >= 0;
        if (served && need > 0 && need_to > count) {
            if (count >= 0) latch_error(a.err, ERR_NO_BLOCKS);
            served = false;
        }
        int64_t taken_all;
        (void)block_scan(served ? need : 0, part, taken_all);
        taken += taken_all;
        if (in) {
            Entry e;
            e.row = served ? r : -1;
            e.held = rec.y;
            e.total = rec.y + (int)need;
            e.base = (int)(count - 1 - (need_to - need));
            e.q0 = (int)min(rows_to - m, (int64_t)INT32_MAX);
            e.rows = m;
            e.ctx = served ? (int)ctx : 0;
            e.tokens = rec.x;
            if (ONE) held[threadIdx.x] = e;
            else a.entries[b] = *reinterpret_cast<TablesEntry*>(&e);
            a.ctx_lens[b] = e.ctx;
            if (b == 0) a.q_start[0] = 0;
            a.q_start[b + 1] = (int)min(rows_to, (int64_t)INT32_MAX);
            if (served && need > 0) reinterpret_cast<int*>(a.requests + r)[1] = e.total;
        }
        rows_before += rows_all;
        need_before += need_all;
    }
    // Those served are the first ones that need blocks, so what they took is a front of the sums.
    if (threadIdx.x == 0 && taken > 0) *a.pool_count = count - (int)taken;
    if (!ONE) return;
    __syncthreads();
    const int n = a.B * a.width;  // small: the host checks
    for (int x = threadIdx.x; x < n; x += kTabThreads) {
        const int b = x / a.width;
        fill_block(a, held[b], b, x - b * a.width);
    }
    if (!a.positions && !a.slots) return;
    for (int i = threadIdx.x; i < a.max_rows; i += kTabThreads) {
        const int b = entry_of_row(a.B, i, [&](int x) -> int64_t { return x < a.B ? held[x].q0 : (int64_t)held[a.B - 1].q0 + held[a.B - 1].rows; });
        fill_row(a, held[max(b, 0)], i, b < 0 ? -1 : i - held[b].q0);
    }
}

__global__ __launch_bounds__(kFillThreads) void tables_fill_kernel(TablesArgs a) {
    const Entry* entries = reinterpret_cast<const Entry*>(a.entries);
    if ((int64_t)blockIdx.x < a.table_wgs) {
        const int chunks = (a.width + kFillEntries - 1) / kFillEntries;
        const int b = (int)(blockIdx.x / chunks), c = (int)(blockIdx.x - (unsigned)b * chunks);
        const Entry e = entries[b];
        const int to = min(a.width, (c + 1) * kFillEntries);
#pragma unroll 4
        for (int i = c * kFillEntries + threadIdx.x; i < to; i += kFillThreads) fill_block(a, e, b, i);
        return;
    }
    const int64_t first = ((int64_t)blockIdx.x - a.table_wgs) * kFillEntries;
    const int64_t to = min((int64_t)a.max_rows, first + kFillEntries);
    for (int64_t i = first + threadIdx.x; i < to; i += kFillThreads) {
        const int b = entry_of_row(a.B, i, [&](int x) -> int64_t { return a.q_start[x]; });
        const Entry e = entries[max(b, 0)];
        fill_row(a, e, i, b < 0 ? -1 : (int)(i - e.q0));
    }
}

// KEEP: the rows that stay of a step; otherwise requests that end, whose blocks tables_free_kernel moves.
template <bool KEEP>
__global__ __launch_bounds__(kTabThreads) void tables_shrink_kernel(TablesArgs a) {
    extern __shared__ uint32_t names_lds[];
    __shared__ int64_t part[kTabWaves];
    __shared__ int to_base[kTabThreads], from_row[kTabThreads], from_at[kTabThreads];
    Names names;
    names.mark(a, names_lds);
    const int count = pool_count(a);
    // What an entry gives back: blocks [stay, held) of request r.
    struct Shrink {
        int r, stay, held, tokens;
    };
    auto look = [&](int b) -> Shrink {
        Shrink s{-1, 0, 0, 0};
        int4 rec;
        s.r = names.request(a, b);
        if (s.r >= 0 && !load_record(a, s.r, rec)) s.r = -1;
        if (s.r < 0) return s;
        s.held = rec.y;
        s.stay = rec.z;
        if (!KEEP) return s;
        const int q0 = a.q_start[b], q1 = a.q_start[b + 1];
        const int64_t m = (int64_t)q1 - q0, c = a.ctx_lens[b];
        int64_t k = m;
        if (m > 0) k = (int64_t)a.kept[b] + a.kept_plus;
        if (q0 < 0 || m < 0 || k < 0 || k > m) {
            latch_error(a.err, ERR_Q_LAYOUT);
            s.r = -1;
        } else if (c < m || c - m + k > (int64_t)rec.y * a.bs) {
            if (c != 0) latch_error(a.err, ERR_CTX_LEN);  // 0: extend left the entry out
            s.r = -1;
        } else {
            s.tokens = (int)(c - m + k);
            s.stay = min(rec.y, max(rec.z, (s.tokens + a.bs - 1) / a.bs));
        }
        return s;
    };
    // First what all give back: a pool that cannot take it leaves everything as it is.
    int64_t all = 0;
    Shrink s{-1, 0, 0, 0};
    for (int b0 = 0; b0 < a.B; b0 += kTabThreads) {
        const int b = b0 + threadIdx.x;
        s = b < a.B ? look(b) : Shrink{-1, 0, 0, 0};
        int64_t total;
        (void)block_scan(s.r >= 0 ? s.held - s.stay : 0, part, total);
        all += total;
    }
    const bool fits = count >= 0 && count + all <= a.pool_cap;
    if (!fits && threadIdx.x == 0) latch_error(a.err, ERR_POOL);
    int64_t before = fits ? count : 0;
    for (int b0 = 0; b0 < a.B; b0 += kTabThreads) {
        const int b = b0 + threadIdx.x;
        if (a.B > kTabThreads) s = b < a.B ? look(b) : Shrink{-1, 0, 0, 0};  // a single strip has it from above
        const bool live = fits && s.r >= 0;
        const int freed = live ? s.held - s.stay : 0;
        int64_t total;
        const int64_t to = before + block_scan(freed, part, total);
        if (b < a.B) {
            if (KEEP) {
                a.out_ctx[b] = live ? s.tokens : 0;
                if (live) *reinterpret_cast<int2*>(a.requests + s.r) = make_int2(s.tokens, s.stay);
            } else {
                Entry e{};
                e.row = live ? s.r : -1;
                e.held = s.stay;
                e.total = s.held;
                e.base = (int)(to - freed);
                a.entries[b] = *reinterpret_cast<TablesEntry*>(&e);
                if (live) a.requests[s.r] = make_int4(0, 0, 0, 0);
            }
        }
        if (KEEP) {
            to_base[threadIdx.x] = (int)(to - freed - before);
            from_row[threadIdx.x] = s.r;
            from_at[threadIdx.x] = s.stay;
            __syncthreads();
            const int strip = min(kTabThreads, a.B - b0);
            for (int64_t x = threadIdx.x; x < total; x += kTabThreads) {
                // The last entry whose blocks start at or before x: those that give none share its start.
                const int t = entry_of_row(strip, x, [&](int y) -> int64_t { return y < strip ? (int64_t)to_base[y] : total; });
                a.pool_out[before + x] = a.blocks[(size_t)from_row[t] * a.state_blocks + from_at[t] + (x - to_base[t])];
            }
            __syncthreads();
        }
        before += total;
    }
    if (threadIdx.x == 0 && fits && all > 0) *a.pool_count = count + (int)all;
}

// The blocks that requests which ended give back.
__global__ __launch_bounds__(kFillThreads) void tables_free_kernel(TablesArgs a) {
    const int chunks = (a.state_blocks + kFillEntries - 1) / kFillEntries;
    const int b = (int)(blockIdx.x / chunks), c = (int)(blockIdx.x - (unsigned)b * chunks);
    const Entry e = reinterpret_cast<const Entry*>(a.entries)[b];
    if (e.row < 0) return;
    const int freed = e.total - e.held, to = min(freed, (c + 1) * kFillEntries);
#pragma unroll 4
    for (int i = c * kFillEntries + threadIdx.x; i < to; i += kFillThreads)
        a.pool_out[e.base + i] = a.blocks[(size_t)e.row * a.state_blocks + e.held + i];
}

size_t names_bytes(const TablesArgs& a) { return (size_t)((a.num_rows + 31) / 32) * 2 * sizeof(uint32_t); }

}  // namespace

bool tables_one_launch(const TablesArgs& a) {
    return a.B <= kTabThreads && names_bytes(a) <= 8192 && (int64_t)a.B * a.width <= kTablesOneEntries && a.max_rows <= kTablesOneRows;
}

int64_t tables_fill_wgs(const TablesArgs& a, int64_t& table_wgs) {
    table_wgs = (int64_t)a.B * ((a.width + kFillEntries - 1) / kFillEntries);
    return table_wgs + (a.positions || a.slots ? ((int64_t)a.max_rows + kFillEntries - 1) / kFillEntries : 0);
}

int64_t tables_free_wgs(const TablesArgs& a) { return (int64_t)a.B * ((a.state_blocks + kFillEntries - 1) / kFillEntries); }

hipError_t launch_tables_extend(const TablesArgs& a0, hipStream_t stream) {
    TablesArgs a = a0;
    if (tables_one_launch(a)) {
        tables_extend_kernel<true><<<dim3(1), kTabThreads, names_bytes(a), stream>>>(a);
        return hipGetLastError();
    }
    tables_extend_kernel<false><<<dim3(1), kTabThreads, names_bytes(a), stream>>>(a);
    const int64_t wgs = tables_fill_wgs(a, a.table_wgs);
    tables_fill_kernel<<<dim3((unsigned)wgs), kFillThreads, 0, stream>>>(a);
    return hipGetLastError();
}

hipError_t launch_tables_keep(const TablesArgs& a, hipStream_t stream) {
    tables_shrink_kernel<true><<<dim3(1), kTabThreads, names_bytes(a), stream>>>(a);
    return hipGetLastError();
}

hipError_t launch_tables_release(const TablesArgs& a, hipStream_t stream) {
    tables_shrink_kernel<false><<<dim3(1), kTabThreads, names_bytes(a), stream>>>(a);
    tables_free_kernel<<<dim3((unsigned)tables_free_wgs(a)), kFillThreads, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace kyro
