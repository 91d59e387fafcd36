// Paged attention for a batch whose sequences share prefixes (block tables that start with the same blocks).
//
// A softmax over a context is the merge of softmaxes over its parts, so the tokens that a group of sequences has in
// common need not be walked once a sequence: all rows of the group, which are consecutive rows of the query, see all
// of them, and become the rows of one product. What remains of each sequence, its own tokens, is walked as before.
//   * attn_shared_plan_kernel: one workgroup checks the groups, decides for each whether its common tokens are worth
//     a pass of their own, and lays the work out on a line: row groups of 128 rows over common tokens, then each
//     sequence's row groups over its own. The line is cut into equal shares, one for each workgroup that the chip
//     holds, so that all have the same to do whatever the lengths; places are sums over the batch.
//   * attn_shared_kernel (shared_attention.hpp) walks a share. With 8 kv heads the dispatcher's round-robin over the 8
//     XCDs keeps every head's K/V in one XCD's L2.
//   * attn_shared_combine_kernel merges each row's partial states, common ones and own ones.
// Three kernels of one call, on MI355X, bf16, 32/8 heads of 128 (us, medians of 20 calls, and what the call has to move or
// multiply):
//   64 sequences of 1 row behind 8192 tokens, 16 to 1000 of their own   5.7 + 36.0 +  5.2   168 MB: 26 at 6.5 TB/s
//   64 of 8 rows behind 4096, 100 to 1500 of their own                  5.9 + 71.1 + 10.5   237 MB: 36, and 41 GFLOP: 35
//   32 of 1 row behind 32768, 20 to 300 of their own                    5.7 + 33.7 +  7.0   156 MB: 24
//   8 of 100 to 300 rows behind 6000                                    6.3 + 204  + 19.5   160 GFLOP: 134 at 1.2 PFLOP/s
// (the last one's first calls, before the clock falls: 177 and 17.4).
// The first and third stream: 4.7 TB/s over the main kernel, whose workgroups' states (64 KiB each, 33 MB) are written and
// read beside that. What bounds the others stands at the loop (shared_attention.hpp).
// Common tokens are taken in whole tiles (64 tokens, 32 in f32 and above head dim 128), so that no tile needs a
// mask at its start; what is left of the last one counts as each sequence's own.
#include "attention_rows.hpp"
#include "common.hpp"
#include "kernels.hpp"

namespace kyro {

namespace {

constexpr int kThreads = 256;

// Tiles up to the last token that row group rg of q_len rows sees.
__device__ __forceinline__ int visible_tiles(const SharedArgs& s, int rg, int q_len, int ctx) {
    const int last = min((rg + 1) * kPrefillRows, q_len * s.a.group) - 1;
    const int vis = s.a.causal ? ctx - q_len + (int)((unsigned)last / (unsigned)s.a.group) + 1 : ctx;
    return (max(vis, 0) + (1 << s.tile_shift) - 1) >> s.tile_shift;
}

__device__ __forceinline__ int row_groups_of(const SharedArgs& s, int rows) {
    return (int)(((uint64_t)(unsigned)rows * (unsigned)s.a.group + kPrefillRows - 1) / kPrefillRows);
}

// A unit of T tiles at `at` on the line whose shares are `share` long: workgroups first .. last hold a piece
// of it, and cut(w) is the tile where the piece of workgroup w + 1 begins. A cut inside the unit's fixed cost, which is at
// its start, is moved to the first tile, and workgroup `first` then has no piece; a share is longer than that cost, so
// that the other cuts lie between tiles and the pieces follow each other.
struct Pieces {
    int at, share, T, first, last;
    __device__ Pieces(int pos, int tiles, int len) : at(pos), share(len), T(tiles) {
        first = (int)((unsigned)at / (unsigned)share);
        last = (int)((unsigned)(end() - 1) / (unsigned)share);
    }
    __device__ int end() const { return at + kSharedUnitCost + T; }
    __device__ int cut(int w) const {
        if (w < first) return 0;
        if (w >= last) return T;
        return max((w + 1) * share - at - kSharedUnitCost, 0);  // below T: workgroup w + 1 begins before end()
    }
    __device__ int first_piece() const { return first + (first < last && cut(first) == 0); }
    __device__ int pieces() const { return last - first_piece() + 1; }
    // Whether the line's share w begins, or ends, in the unit.
    __device__ bool begins(int w) const { return w * share >= at; }
    __device__ bool ends(int w, int line) const { return w < last || (w + 1) * share == end() || end() == line; }
};

// One workgroup of N threads lists the work: thread i has sequence i, group i and the sequences' own unit i, and goes on
// with i + N, .. in the form for any batch (!ONE), whose records are in scratch; ONE holds them in LDS. It runs on one CU
// while the others wait, and most of its time is the latency of what follows from each other, and of fetching code that
// runs once: loads are issued together, barriers are few, sums are of 32 bits, and nothing is divided that a
// shift does. 5.6 to 6.9 us for the batches of 8 to 128 sequences below, where a form with a loop over each sequence's
// row groups and sums of 64 bits took 9 to 20.
template <int N, bool ONE>
__global__ __launch_bounds__(N) void attn_shared_plan_kernel(SharedArgs s) {
    const AttnArgs& a = s.a;
    constexpr int kHeld = ONE ? N : 1;
    __shared__ uint32_t part[2 * 3 * (N / 64)];
    __shared__ int l_starts[kHeld + 1], l_rows[kHeld + 1], l_base[kHeld];
    __shared__ int4 l_seqs[kHeld], l_units[kHeld];
    __shared__ int2 l_counts[kHeld], l_places[kHeld];
    __shared__ int l_blocks[kHeld], l_firsts[kHeld], bad_groups;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int32_t* const starts = ONE ? l_starts : s.group_starts;     // first sequences of the groups
    int4* const seqs = ONE ? l_seqs : s.seqs;                          // {first row, rows, context length, group or -1}
    int2* const counts = ONE ? l_counts : s.counts;                    // {sequences that share, their row groups}
    int2* const places = ONE ? l_places : s.places;                    // {place on the line, first unit or -1}
    int* const base = ONE ? l_base : s.bases;                          // first own unit
    int* const firsts = ONE ? l_firsts : s.firsts;                     // first sequence that shares
    BlockSums<N, 3> sums{part};
    auto each = [&](int n, auto&& f) {
        if constexpr (ONE) {
            if (t < n) f(t);
        } else {
            for (int i = t; i < n; i += N) f(i);
        }
    };
    auto q_row = [&](int b) -> int { return ONE ? l_rows[b] : a.q_start ? a.q_start[b] : b; };

    if (t == 0) bad_groups = 0;
    __syncthreads();
    each(max(a.B, s.G), [&](int i) {
        const int b = min(i, a.B - 1), g = min(i, s.G - 1);
        const int64_t c = a.ctx_lens[b];
        const int q0 = a.q_start ? a.q_start[b] : b, q1 = a.q_start ? a.q_start[b + 1] : b + 1;
        const int s0 = s.group_starts[g], s1 = s.group_starts[g + 1], nb = s.group_blocks[g];
        int err = 0;
        if (i < a.B) {
            if (c < 0 || c > (int64_t)a.max_blocks * a.bs) err |= ERR_CTX_LEN;
            if (q0 < 0 || q1 < q0 || q1 > a.total_q || q1 - q0 > a.max_q_len) err |= ERR_Q_LAYOUT;
            seqs[b] = make_int4(q0, err ? 0 : q1 - q0, err ? 0 : (int)c, -1);
            if (ONE) {
                l_rows[b] = q0;
                if (b == a.B - 1) l_rows[a.B] = q1;
            }
        }
        if (i < s.G) {
            if (s0 < 0 || s1 < s0 || s1 > a.B) bad_groups = 1;
            if (nb < 0 || nb > a.max_blocks) err |= ERR_GROUPS;
            counts[g] = make_int2(0, 0);
            firsts[g] = INT32_MAX;
            if (ONE) {
                l_starts[g] = s0;
                l_blocks[g] = nb;
                if (g == s.G - 1) l_starts[s.G] = s1;
            }
        }
        if (err) latch_error(a.err, err);
    });
    __syncthreads();
    const int G = bad_groups ? 0 : s.G;
    if (G == 0 && t == 0) latch_error(a.err, ERR_GROUPS);

    // {first row, rows, common tiles} of a group; no tiles where its numbers are wrong.
    auto group_of = [&](int g) -> int3 {
        const int nb = ONE ? l_blocks[g] : s.group_blocks[g], q0 = q_row(starts[g]), q1 = q_row(starts[g + 1]);
        const bool ok = nb > 0 && nb <= a.max_blocks && q0 >= 0 && q0 <= q1 && q1 <= a.total_q;
        return ok ? make_int3(q0, q1 - q0, (nb * a.bs) >> s.tile_shift) : make_int3(0, 0, 0);
    };
    // The last of n ascending values that is at most x, or -1.
    auto last_at_most = [](const int* from, int n, int x) -> int {
        int lo = 0, hi = n;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (from[mid] <= x) lo = mid + 1;
            else hi = mid;
        }
        return lo - 1;
    };
    // The group that a sequence shares with, if every row of it sees the common tokens.
    each(G > 0 ? a.B : 0, [&](int b) {
        const int4 e = seqs[b];
        const int g = last_at_most(starts, G, b);
        if (e.y == 0 || g < 0 || b >= starts[g + 1]) return;
        const int3 gr = group_of(g);
        const int sees = a.causal ? e.z - e.y + 1 : e.z;
        if (gr.z > 0 && sees >= gr.z << s.tile_shift && e.x >= gr.x && e.x + e.y <= gr.x + gr.y) {
            seqs[b].w = g;
            atomicAdd(&counts[g].x, 1);
            atomicAdd(&counts[g].y, row_groups_of(s, e.y));
            atomicMin(&firsts[g], b);
        }
    });
    if (!ONE) __threadfence();  // atomics on scratch
    // Own units: one a sequence where no sequence has more, also for one without rows.
    int units = a.B;
    if (a.row_groups > 1) {
        uint32_t before = 0;
        for (int b0 = 0; b0 < a.B; b0 += N) {
            const int b = b0 + t;
            uint32_t x[1] = {b < a.B ? (uint32_t)row_groups_of(s, seqs[b].y) : 0}, all[1];
            const uint32_t n = x[0];
            sums.scan(x, all);
            if (b < a.B) base[b] = (int)min(add_sat(before, x[0] - n), (uint32_t)INT32_MAX);
            before = add_sat(before, all[0]);
            if (ONE) break;
        }
        units = (int)min(before, (uint32_t)INT32_MAX);
    }
    const bool crowded = units > s.own_cap;  // ranges that overlap around an invalid one
    if (crowded) units = 0;
    __syncthreads();

    // The line: the common units of all groups, then the own units. A group shares where the tiles it saves are worth the
    // states it adds.
    auto shares = [&](int g, int3& gr) -> bool {
        gr = group_of(g);
        const int2 k = counts[g];
        const int rgs = row_groups_of(s, gr.y);
        return k.x > 1 && (int64_t)(k.y - rgs) * gr.z > (int64_t)(k.y + rgs) * s.merge_cost;
    };
    uint32_t common_line = 0, common_units = 0, own_line = 0;
    for (int i0 = 0; i0 < max(G, units); i0 += N) {
        const int i = i0 + t;
        uint32_t x[3] = {0, 0, 0}, all[3];
        int4 unit;
        int3 gr;
        if (i < G && shares(i, gr)) {
            x[1] = (uint32_t)row_groups_of(s, gr.y);
            x[0] = (uint32_t)min((uint64_t)x[1] * (uint32_t)(gr.z + kSharedUnitCost), (uint64_t)UINT32_MAX);
        }
        if (i < units) {
            const int b = a.row_groups > 1 ? last_at_most(base, a.B, i) : i;
            const int4 e = seqs[b];
            const int rg = a.row_groups > 1 ? i - base[b] : 0;
            const int first = e.w >= 0 && shares(e.w, gr) ? gr.z : 0;
            unit = make_int4(0, e.y > 0 ? visible_tiles(s, rg, e.y, e.z) - first : -1, b, first);
            if (e.y > 0) x[2] = (uint32_t)(unit.y + kSharedUnitCost);
        }
        const uint32_t len = x[0], n = x[1], own = x[2];
        sums.scan(x, all);
        if (i < G) places[i] = make_int2((int)add_sat(common_line, x[0] - len), n ? (int)add_sat(common_units, x[1] - n) : -1);
        if (i < units) {
            unit.x = (int)add_sat(own_line, x[2] - own);
            (ONE ? l_units[i] : s.merges[2 * i]) = unit;
        }
        common_line = add_sat(common_line, all[0]);
        common_units = add_sat(common_units, all[1]);
        own_line = add_sat(own_line, all[2]);
        if (ONE) break;
    }
    const uint64_t line = (uint64_t)common_line + own_line;
    const uint32_t share = max((uint32_t)((min(line, (uint64_t)INT32_MAX) + s.lanes - 1)) / (uint32_t)s.lanes,
                               (uint32_t)kSharedLeastShare);
    const int whole = (int)line;
    // More than was sized, which valid ranges cannot be: latch it and run nothing.
    const bool over = crowded || common_units > (uint32_t)s.common_cap || line + share > INT32_MAX;
    if (t == 0) {
        if (over) latch_error(a.err, ERR_PLAN);
        s.head[0] = over ? 0 : (int)((whole + share - 1) / share);
        s.head[1] = over ? 0 : units;
    }
    if (over) return;
    if (!ONE || G > 0) __syncthreads();  // places
    // Workgroup w's piece of unit u; an empty unit begins and ends no share.
    auto put = [&](const Pieces& p, int u, int w, const int4& e0, const int4& e1, bool some = true) {
        s.list[2 * (u + w)] = e0;
        s.list[2 * (u + w) + 1] = e1;
        if (some && p.begins(w)) {
            s.starts[3 * w].x = u;
            s.starts[3 * w + 1] = e0;
            s.starts[3 * w + 2] = e1;
        }
        if (some && p.ends(w, whole)) s.starts[3 * w].y = u;
    };
    for (int g = wave; g < G; g += N / 64) {
        const int2 place = places[g];
        if (place.y < 0) continue;
        const int3 gr = group_of(g);
        const int len = gr.z + kSharedUnitCost, rgs = row_groups_of(s, gr.y);
        const int most = (int)((unsigned)(len - 1) / share) + 2;  // pieces of a unit at most
        for (int x = lane; x < rgs * most; x += 64) {
            const int r = (int)((unsigned)x / (unsigned)most), u = place.y + r;
            const Pieces p(place.x + r * len, gr.z, (int)share);
            const int w = p.first + (x - r * most);
            if (x == r * most) s.common_parts[u] = make_int2(u + p.first_piece(), p.pieces());
            if (w > p.last) continue;
            const int from = p.cut(w - 1), to = p.cut(w);
            put(p, u, w, make_int4(from < to ? firsts[g] : -1, gr.x, gr.y, gr.z << s.tile_shift),
                make_int4(r * kPrefillRows, from, (to - from) | kSharedAll, u + w));
        }
    }
    // The sequences' own units, and which row groups are merged.
    each(units, [&](int v) {
        const int4 unit = ONE ? l_units[v] : s.merges[2 * v];
        const int4 e = seqs[unit.z];
        const int row = a.row_groups > 1 ? (v - base[unit.z]) * kPrefillRows : 0, first = unit.w;
        const int u = (int)common_units + v;
        Pieces p((int)common_line + unit.x, max(unit.y, 0), (int)share);
        if (unit.y < 0) p.last = p.first;
        const int pieces = p.pieces();
        const bool parked = unit.y >= 0 && (first > 0 || pieces > 1), none = unit.y < 0 || (first > 0 && p.T == 0);
        for (int w = p.first; w <= p.last; ++w) {
            const int from = p.cut(w - 1), to = p.cut(w);
            const bool piece = !none && (from < to || (p.T == 0 && w == p.last));
            put(p, u, w, make_int4(piece ? unit.z : -1, e.x, e.y, e.z), make_int4(row, first + from, to - from, parked ? v + w : -1),
                unit.y >= 0);
        }
        const int3 gr = first > 0 ? group_of(e.w) : make_int3(0, 0, 0);
        s.merges[2 * v] = make_int4(e.x, parked ? e.y : 0, row, (e.x - gr.x) * a.group + row);
        s.merges[2 * v + 1] = make_int4(v + p.first_piece(), none ? 0 : pieces, first > 0 ? places[e.w].y : -1, 0);
    });
}

// Merges the partial states of the listed row groups. A workgroup takes a slice of one row group's (row, four
// columns) for one kv head, rows fastest, so that the lanes read the neighbouring rows that a state keeps together.
// WAYS of its threads share one such item's states: where items are few, states are many (a row of 32 sequences behind 32768
// tokens with 8 kv heads has 64: 6.8 us for 11.0; one of 8 sequences of 8 rows with one kv head has more than 100, and the
// whole call takes 33 us for 47). With the 524288 items of 64 sequences of 32 rows there are workgroups enough, and
// four threads an item take 14.0 for 10.5.
template <int DR, int WAYS>
__global__ __launch_bounds__(kThreads) void attn_shared_combine_kernel(SharedArgs s) {
    const AttnArgs& a = s.a;
    constexpr int DT = (DR + 31) / 32, Q = DR / 4, kItems = kThreads / WAYS;
    __shared__ float merged[WAYS > 1 ? WAYS - 1 : 1][6][kItems];
    const int item = (int)threadIdx.x % kItems, way = (int)threadIdx.x / kItems;
    const int entry = (int)blockIdx.x / a.Hkv, kvh = (int)blockIdx.x - entry * a.Hkv;
    const int used = s.head[1];
    const int4 e = s.merges[2 * entry], f = s.merges[2 * entry + 1];
    if (entry >= used) return;
    const int rows = min(kPrefillRows, e.y * a.group - e.z);
    if (rows <= 0) return;
    const int x = (int)blockIdx.y * kItems + item;
    if (WAYS == 1 && x >= rows * Q) return;
    const bool some = x < rows * Q;
    const int c = some ? x / rows : 0, r = some ? x - c * rows : 0;  // columns 4 c .. 4 c + 3 of row e.z + r
    const int dt = c / 8, k = c / 2 % 4, h = c % 2;
    // The row's partial states: `common` ones over common tokens, then own ones.
    size_t at_common = 0;
    int common = 0, col = r & 31;
    const int own_col = col;
    if (f.z >= 0) {
        const int g = e.w + r;  // the row in its group
        const int2 parts = s.common_parts[f.z + g / kPrefillRows];
        at_common = ((size_t)parts.x * a.Hkv + kvh) * 4 + g % kPrefillRows / 32;
        common = parts.y;
        col = g & 31;
    }
    const size_t at_own = (size_t)s.tail_base + ((size_t)f.x * a.Hkv + kvh) * s.tail_waves + r / 32;
    const int n = common + f.y;
    float M = kNegInf, L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    // States whose loads are in flight; an index past the last reads the last one again, with weight 0. More threads on a CU
    // are worth more than more loads of each: 8 took 28 us for 23 of 1600 prompt rows, and 20 for 17 of 128 requests,
    // though 9 for 11 where 128 rows have 64 states each.
    constexpr int kBatch = 4;
    for (int i0 = way * kBatch; i0 < n; i0 += WAYS * kBatch) {
        float m[kBatch], l[kBatch];
        float4 v[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int x = min(i0 + i, n - 1);
            const size_t wv = x < common ? at_common + (size_t)x * a.Hkv * 4 : at_own + (size_t)(x - common) * a.Hkv * s.tail_waves;
            const int y = x < common ? col : own_col;
            m[i] = a.ws_m[wv * 32 + y];
            l[i] = a.ws_l[wv * 32 + y];
            v[i] = reinterpret_cast<const float4*>(a.ws_acc)[((wv * DT + dt) * 4 + k) * 64 + 32 * h + y];
        }
        float mb = M;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) mb = fmaxf(mb, m[i]);
        const float mref = mb == kNegInf ? 0.f : mb;
        const float old = fast_exp2(M - mref);
        L *= old;
        o.x *= old;
        o.y *= old;
        o.z *= old;
        o.w *= old;
        M = mb;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const float w = i0 + i < n ? fast_exp2(m[i] - mref) : 0.f;
            L += w * l[i];
            o.x += w * v[i].x;
            o.y += w * v[i].y;
            o.z += w * v[i].z;
            o.w += w * v[i].w;
        }
    }
    if constexpr (WAYS > 1) {
        if (way > 0) {
            const float held[6] = {M, L, o.x, o.y, o.z, o.w};
#pragma unroll
            for (int k = 0; k < 6; ++k) merged[way - 1][k][item] = held[k];
        }
        __syncthreads();
        if (way > 0 || !some) return;
        float mb = M;
#pragma unroll
        for (int w = 0; w < WAYS - 1; ++w) mb = fmaxf(mb, merged[w][0][item]);
        const float mref = mb == kNegInf ? 0.f : mb;
        const float old = fast_exp2(M - mref);
        L *= old, o.x *= old, o.y *= old, o.z *= old, o.w *= old;
#pragma unroll
        for (int w = 0; w < WAYS - 1; ++w) {
            const float f = fast_exp2(merged[w][0][item] - mref);
            L += f * merged[w][1][item];
            o.x += f * merged[w][2][item];
            o.y += f * merged[w][3][item];
            o.z += f * merged[w][4][item];
            o.w += f * merged[w][5][item];
        }
    }
    const float inv = L > 0.f ? 1.f / L : 0.f;
    SeqInfo si;
    si.q0 = e.x;
    si.kvh = kvh;
    store_row4<DR>(a, out_row(a, si, e.z + r), 4 * c, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

constexpr long long kSharedFewItems = 1 << 18;  // of all row groups: up to so many, four threads an item

template <int DR>
void launch_combine(const SharedArgs& s, hipStream_t stream) {
    const AttnArgs& a = s.a;
    const int rows = a.rows_cap < kPrefillRows ? a.rows_cap : kPrefillRows, items = rows * (DR / 4);
    const unsigned groups = (unsigned)((long long)s.own_cap * a.Hkv);
    if ((long long)groups * items <= kSharedFewItems) attn_shared_combine_kernel<DR, 4><<<dim3(groups, (unsigned)((items + 63) / 64)), kThreads, 0, stream>>>(s);
    else attn_shared_combine_kernel<DR, 1><<<dim3(groups, (unsigned)((items + kThreads - 1) / kThreads)), kThreads, 0, stream>>>(s);
}

}  // namespace

hipError_t launch_shared_bf16(const SharedArgs& s, hipStream_t stream);
hipError_t launch_shared_wide(const SharedArgs& s, hipStream_t stream);
hipError_t launch_shared_f32(const SharedArgs& s, hipStream_t stream);

hipError_t launch_attention_shared(const SharedArgs& s, hipStream_t stream) {
    const AttnArgs& a = s.a;
    if (a.B <= 256 && s.G <= 256 && s.own_cap <= 256) attn_shared_plan_kernel<256, true><<<dim3(1), 256, 0, stream>>>(s);
    else attn_shared_plan_kernel<1024, false><<<dim3(1), 1024, 0, stream>>>(s);
    const hipError_t e = !a.dtype_bf16 ? launch_shared_f32(s, stream) : a.D > 128 ? launch_shared_wide(s, stream) : launch_shared_bf16(s, stream);
    if (e != hipSuccess) return e;
    switch (a.D) {
        case 64: launch_combine<64>(s, stream); break;
        case 80: launch_combine<80>(s, stream); break;
        case 96: launch_combine<96>(s, stream); break;
        case 112: launch_combine<112>(s, stream); break;
        case 128: launch_combine<128>(s, stream); break;
        case 160: launch_combine<160>(s, stream); break;
        case 192: launch_combine<192>(s, stream); break;
        case 224: launch_combine<224>(s, stream); break;
        case 256: launch_combine<256>(s, stream); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace kyro
