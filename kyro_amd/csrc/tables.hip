// Block tables, row ranges and cache slots of a step from the requests' own records, and the pool of free
// blocks (include/kyro_tables.h).
//
// Everything that depends on the order of the batch (rows before an entry, blocks taken or given back before it)
// is a prefix sum over the batch, so one workgroup works the batch out, 1024 entries at a time: it reads each
// entry's state row and record, checks them, scans rows and blocks, and updates records and pool count. What is
// left has no order: table rows, positions and slots are written by as many workgroups as they fill
// (tables_fill_kernel), or, where they are few, by the first one right away, which saves the second launch.
//
// What bounds it: latency. One request: 5.4 us, 64 with tables of 264 blocks and 8 rows each: 11.7 in one launch (6.7 + 3.6
// in two, and 3.4 more of the host), both no more than the call from Python (11.6). 264 entries with tables of 8192 blocks,
// 28 MB to move: 5.7 + 9.5, the second at 2.9 TB/s. Rows that stay: 5.6 us for 64 requests that give 23 blocks back, 10.1
// for 1024 that give 1898. Requests that end: 3.3 + 2.6 for 64 of 110 blocks each, 3.7 + 6.6 for 256 of 1580. All these on a
// state that is put back before each call, so that blocks move; a repeated call, which moves none, takes 4.8, 10.7, 4.2 +
// 8.6, 3.8 and 7.1.
#include "common.hpp"

namespace kyro {

namespace {

constexpr int kTabThreads = 1024;
constexpr int kTabWaves = kTabThreads / 64;
constexpr int kFillThreads = 256;
constexpr int kFillEntries = 2048;  // table entries or freed blocks of one fill workgroup
static_assert(kTablesMaxWidth + (int64_t)kFillEntries <= (int64_t)INT32_MAX + 1, "ends of workgroups in 32 bits");
constexpr int kFillRows = 512;      // rows of one fill workgroup: what a row reads follows from what it read before

// What the scan hands to the fill, for each entry of the batch.
struct Entry {
    int row, held, total, base;  // request (-1: left out); blocks before and after; pool entry of the first
                                 // block taken (going down) or given back (going up)
    int q0, rows, ctx, tokens;   // its rows, context length with them, tokens before them
};
static_assert(sizeof(Entry) == kTablesEntryBytes, "scratch of an entry");

// The batch's state rows, checked: marks in LDS which requests are named, and which twice.
struct Names {
    uint32_t* once;   // bits of requests named
    uint32_t* twice;  // named again

    // `mine` is the state row of entry threadIdx.x, which the caller has loaded.
    __device__ void mark(const TablesArgs& a, uint32_t* lds, int mine) {
        const int words = (a.num_rows + 31) / 32;
        once = lds;
        twice = lds + words;
        for (int i = threadIdx.x; i < 2 * words; i += kTabThreads) lds[i] = 0;
        __syncthreads();
        for (int b = threadIdx.x; b < a.B; b += kTabThreads) {
            const int r = b < kTabThreads ? mine : state_row(a, b);
            if (r < 0 || r >= a.num_rows) continue;
            const uint32_t bit = 1u << (r & 31);
            if (atomicOr(&once[r >> 5], bit) & bit) atomicOr(&twice[r >> 5], bit);
        }
        __syncthreads();
    }

    static __device__ int state_row(const TablesArgs& a, int b) { return a.state_rows ? a.state_rows[b] : b; }

    // Request of an entry with state row r, or -1 for padding and for one that is not (latched).
    __device__ int request(const TablesArgs& a, int r) const {
        if (r < 0) return -1;
        if (r >= a.num_rows || ((twice[r >> 5] >> (r & 31)) & 1u)) {
            latch_error(a.err, ERR_STATE_ROW);
            return -1;
        }
        return r;
    }
};

// The record {tokens, held, shared, -} of state row r where there is one.
__device__ __forceinline__ int4 load_record(const TablesArgs& a, int r) {
    return r >= 0 && r < a.num_rows ? a.requests[r] : make_int4(0, 0, 0, 0);
}

// False (latched) where a record's numbers do not fit each other.
__device__ __forceinline__ bool check_record(const TablesArgs& a, const int4& rec) {
    const bool ok = rec.x >= 0 && rec.z >= 0 && rec.z <= rec.y && rec.y <= a.state_blocks &&
                    (int64_t)rec.x <= (int64_t)rec.y * a.bs;
    if (!ok) latch_error(a.err, ERR_REQUEST);
    return ok;
}

// The pool's count, or -1 (latched) where it is none.
__device__ __forceinline__ int check_count(const TablesArgs& a, int n) {
    if (n >= 0 && n <= a.pool_cap) return n;
    if (threadIdx.x == 0) latch_error(a.err, ERR_POOL);
    return -1;
}

// Entries i, i + stride, .. below `to` of the table row of entry e; a block that is new is the request's from now on. The
// loads of kFillBatch entries are in flight together: one without a block loads what is there anyway.
constexpr int kFillBatch = 8;
__device__ __forceinline__ void fill_blocks(const TablesArgs& a, const Entry& e, int b, int i, int to, int stride) {
    int64_t* own = a.blocks + (size_t)max(e.row, 0) * a.state_blocks;
    int64_t* table = a.table + (size_t)b * a.width;
    const int total = e.row >= 0 ? e.total : 0;
    for (; i < to; i += kFillBatch * stride) {
        int64_t id[kFillBatch];
#pragma unroll
        for (int k = 0; k < kFillBatch; ++k) {
            const int x = i + k * stride;
            const int64_t* from = x < total && x >= e.held ? a.pool + (e.base - (x - e.held)) : own + (x < total ? x : 0);
            id[k] = *from;
        }
#pragma unroll
        for (int k = 0; k < kFillBatch; ++k) {
            const int x = i + k * stride;
            if (x >= to) continue;
            if (x < total && (id[k] < 0 || id[k] >= a.num_blocks)) latch_error(a.err, ERR_BLOCK_ID);
            if (x < total && x >= e.held) own[x] = id[k];
            table[x] = x < total ? id[k] : 0;
        }
    }
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

// ONE: the whole call (at most kTabThreads entries). A wave fills a table row, or several of them that are short: 375 rows
// of 6 blocks took 34.8 us a call with one row a wave; now such calls are bound by the host like the others.
template <bool ONE>
__global__ __launch_bounds__(kTabThreads) void tables_extend_kernel(TablesArgs a) {
    extern __shared__ uint32_t names_lds[];
    __shared__ uint32_t part[2 * 2 * kTabWaves];
    __shared__ int taken;  // blocks that the entries served take
    __shared__ Entry held[ONE ? kTabThreads : 1];
    struct Item {
        int r, m;
        int4 rec;
    };
    auto load = [&](int b) -> Item {
        Item x{-1, 0, make_int4(0, 0, 0, 0)};
        if (b >= a.B) return x;
        x.r = Names::state_row(a, b);
        x.m = a.new_rows[b];
        x.rec = load_record(a, x.r);
        return x;
    };
    const int in_pool = *a.pool_count;
    Item x = load(threadIdx.x);
    if (threadIdx.x == 0) taken = 0;
    Names names;
    names.mark(a, names_lds, x.r);
    const int count = check_count(a, in_pool);
    BlockSums<kTabThreads, 2> sums{part};
    uint32_t rows_before = 0, need_before = 0;
    for (int b0 = 0; b0 < a.B; b0 += kTabThreads) {
        const int b = b0 + threadIdx.x;
        if (b0 > 0) x = load(b);
        int r = b < a.B ? names.request(a, x.r) : -1, m = x.m;
        if (m < 0) {
            latch_error(a.err, ERR_Q_LAYOUT);
            m = 0;
            r = -1;
        }
        if (r >= 0 && !check_record(a, x.rec)) r = -1;
        const int64_t ctx = (int64_t)x.rec.x + m;
        const bool long_ = ctx > (int64_t)min(a.width, a.state_blocks) * a.bs;
        const int need = r >= 0 && !long_ ? max((int)((ctx + a.bs - 1) / a.bs) - x.rec.y, 0) : 0;
        // Rows and blocks of the batch up to here. Entries past max_rows are left out, and so are all that follow, so
        // that what they would need counts against none that is served.
        uint32_t to[2] = {(uint32_t)m, (uint32_t)need}, all[2];
        sums.scan(to, all);
        const uint32_t rows_to = add_sat(rows_before, to[0]), need_to = add_sat(need_before, to[1]);
        if (r >= 0 && rows_to > (uint32_t)a.max_rows) {
            latch_error(a.err, ERR_Q_LAYOUT);
            r = -1;
        }
        if (r >= 0 && long_) {
            latch_error(a.err, ERR_CTX_LEN);
            r = -1;
        }
        if (r >= 0 && need > 0 && (count < 0 || need_to > (uint32_t)count)) {
            if (count >= 0) latch_error(a.err, ERR_NO_BLOCKS);
            r = -1;
        }
        if (b < a.B) {
            Entry e;
            e.row = r;
            e.held = x.rec.y;
            e.total = x.rec.y + need;
            e.base = count - 1 - (int)(need_to - need);
            e.q0 = (int)min(rows_to - m, (uint32_t)INT32_MAX);
            e.rows = m;
            e.ctx = r >= 0 ? (int)ctx : 0;
            e.tokens = x.rec.x;
            if (ONE) held[threadIdx.x] = e;
            else a.entries[b] = *reinterpret_cast<TablesEntry*>(&e);
            a.ctx_lens[b] = e.ctx;
            if (b == 0) a.q_start[0] = 0;
            a.q_start[b + 1] = (int)min(rows_to, (uint32_t)INT32_MAX);
            if (r >= 0 && need > 0) {
                reinterpret_cast<int*>(a.requests + r)[1] = e.total;
                atomicMax(&taken, (int)need_to);  // those served are the first ones that need blocks
            }
        }
        rows_before = add_sat(rows_before, all[0]);
        need_before = add_sat(need_before, all[1]);
    }
    __syncthreads();
    if (threadIdx.x == 0 && taken > 0) *a.pool_count = count - taken;
    if (!ONE) return;
    int shift = 0;  // log2 of a row's lanes
    while (shift < 6 && kFillBatch << shift < a.width) ++shift;
    for (int b = threadIdx.x >> shift; b < a.B; b += kTabThreads >> shift)
        fill_blocks(a, held[b], b, threadIdx.x & ((1 << shift) - 1), a.width, 1 << shift);
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
        fill_blocks(a, e, b, c * kFillEntries + threadIdx.x, min(a.width, (c + 1) * kFillEntries), kFillThreads);
        return;
    }
    // The entries of the workgroup's rows, whose starts it takes to LDS unless many without rows lie between them.
    __shared__ int starts[kFillRows + 2];
    const int64_t first = ((int64_t)blockIdx.x - a.table_wgs) * kFillRows;
    const int64_t to = min((int64_t)a.max_rows, first + kFillRows);
    auto start = [&](int x) -> int64_t { return a.q_start[x]; };
    const int64_t rows = start(a.B);
    const int from = max(entry_of_row(a.B, first, start), 0);
    const int n = rows <= first ? 0 : entry_of_row(a.B, min(to, rows) - 1, start) - from + 1;
    const bool held = n <= kFillRows;
    if (held) {
        for (int x = threadIdx.x; x <= n; x += kFillThreads) starts[x] = a.q_start[from + x];
        __syncthreads();
    }
    for (int64_t i = first + threadIdx.x; i < to; i += kFillThreads) {
        int b = -1;
        if (i < rows) b = held ? from + entry_of_row(n, i, [&](int x) -> int64_t { return starts[x]; }) : entry_of_row(a.B, i, start);
        const Entry e = entries[max(b, 0)];
        fill_row(a, e, i, b < 0 ? -1 : (int)(i - e.q0));
    }
}

// KEEP: the rows that stay of a step; otherwise requests that end, whose blocks tables_free_kernel moves.
template <bool KEEP>
__global__ __launch_bounds__(kTabThreads) void tables_shrink_kernel(TablesArgs a) {
    extern __shared__ uint32_t names_lds[];
    __shared__ uint32_t part[2 * kTabWaves];
    __shared__ int to_base[kTabThreads], from_row[kTabThreads], from_at[kTabThreads];
    struct Item {
        int r, q0, q1, kept;
        int64_t c;
        int4 rec;
    };
    auto load = [&](int b) -> Item {
        Item x{-1, 0, 0, 0, 0, make_int4(0, 0, 0, 0)};
        if (b >= a.B) return x;
        x.r = Names::state_row(a, b);
        if (KEEP) {
            x.q0 = a.q_start[b];
            x.q1 = a.q_start[b + 1];
            x.kept = a.kept[b];
            x.c = a.ctx_lens[b];
        }
        x.rec = load_record(a, x.r);
        return x;
    };
    const int in_pool = *a.pool_count;
    const Item mine = load(threadIdx.x);
    Names names;
    names.mark(a, names_lds, mine.r);
    const int count = check_count(a, in_pool);
    // What an entry gives back: blocks [stay, held) of request r.
    struct Shrink {
        int r, stay, held, tokens;
    };
    auto look = [&](int b) -> Shrink {
        Shrink s{-1, 0, 0, 0};
        if (b >= a.B) return s;
        const Item x = b < kTabThreads ? mine : load(b);
        s.r = names.request(a, x.r);
        if (s.r >= 0 && !check_record(a, x.rec)) s.r = -1;
        if (s.r < 0) return s;
        s.held = x.rec.y;
        s.stay = x.rec.z;
        if (!KEEP) return s;
        const int64_t m = (int64_t)x.q1 - x.q0;
        const int64_t k = m > 0 ? (int64_t)x.kept + a.kept_plus : m;
        if (x.q0 < 0 || m < 0 || k < 0 || k > m) {
            latch_error(a.err, ERR_Q_LAYOUT);
            s.r = -1;
        } else if (x.c == 0) {
            s.r = -1;  // extend left the entry out, with rows or none, or the request is empty and brings none
        } else if (x.c < m || x.c - m + k > (int64_t)x.rec.y * a.bs) {
            latch_error(a.err, ERR_CTX_LEN);
            s.r = -1;
        } else {
            s.tokens = (int)(x.c - m + k);
            // Both are below 2^31, their sum below 2^32.
            s.stay = min(x.rec.y, max(x.rec.z, (int)(((unsigned)s.tokens + (unsigned)a.bs - 1u) / (unsigned)a.bs)));
        }
        return s;
    };
    // First what all give back: a pool that cannot take it leaves everything as it is.
    BlockSums<kTabThreads, 1> sums{part};
    uint32_t all = 0, to[1], total[1];
    Shrink s{-1, 0, 0, 0};
    for (int b0 = 0; b0 < a.B; b0 += kTabThreads) {
        s = look(b0 + threadIdx.x);
        to[0] = s.r >= 0 ? (uint32_t)(s.held - s.stay) : 0;
        sums.scan(to, total);
        all = add_sat(all, total[0]);
    }
    const bool fits = count >= 0 && (uint64_t)count + all <= (uint64_t)a.pool_cap;
    if (!fits && threadIdx.x == 0) latch_error(a.err, ERR_POOL);
    int before = fits ? count : 0;
    for (int b0 = 0; b0 < a.B; b0 += kTabThreads) {
        const int b = b0 + threadIdx.x;
        if (a.B > kTabThreads) {  // a single strip has it from above
            s = look(b);
            to[0] = s.r >= 0 ? (uint32_t)(s.held - s.stay) : 0;
            sums.scan(to, total);
        }
        const bool live = fits && s.r >= 0;
        const int base = (int)(to[0] - (s.r >= 0 ? (uint32_t)(s.held - s.stay) : 0));  // behind `before`
        if (b < a.B) {
            if (KEEP) {
                a.out_ctx[b] = live ? s.tokens : 0;
                if (live) *reinterpret_cast<int2*>(a.requests + s.r) = make_int2(s.tokens, s.stay);
            } else {
                Entry e{};
                e.row = live ? s.r : -1;
                e.held = s.stay;
                e.total = s.held;
                e.base = before + base;
                a.entries[b] = *reinterpret_cast<TablesEntry*>(&e);
                if (live) a.requests[s.r] = make_int4(0, 0, 0, 0);
            }
        }
        if (!fits) continue;
        if (KEEP && total[0] > 0) {
            to_base[threadIdx.x] = base;
            from_row[threadIdx.x] = s.r;
            from_at[threadIdx.x] = s.stay;
            __syncthreads();
            const int strip = min(kTabThreads, a.B - b0);
            for (int64_t x = threadIdx.x; x < total[0]; x += kTabThreads) {
                // The last entry whose blocks start at or before x: those that give none share its start.
                const int t = entry_of_row(strip, x, [&](int y) -> int64_t { return y < strip ? (int64_t)to_base[y] : total[0]; });
                a.pool_out[before + x] = a.blocks[(size_t)from_row[t] * a.state_blocks + from_at[t] + (x - to_base[t])];
            }
            __syncthreads();
        }
        before += (int)total[0];
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
    return table_wgs + (a.positions || a.slots ? ((int64_t)a.max_rows + kFillRows - 1) / kFillRows : 0);
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
