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
// Common tokens are taken in whole tiles (64 tokens, 32 in f32 and above head dim 128), so that no tile needs a
// mask at its start; what is left of the last one counts as each sequence's own.
#include "attention_rows.hpp"
#include "common.hpp"
#include "kernels.hpp"

namespace kyro {

namespace {

constexpr int kThreads = 256;

// Tiles up to the last token that row group rg of q_len rows sees, or -1 where it has no rows.
__device__ __forceinline__ int visible_tiles(const SharedArgs& s, int rg, int q_len, int ctx) {
    const int rows = q_len * s.a.group;
    if (rg * kPrefillRows >= rows) return -1;
    const int last = min((rg + 1) * kPrefillRows, rows) - 1;
    const int vis = s.a.causal ? ctx - q_len + last / s.a.group + 1 : ctx;
    return (max(vis, 0) + s.tile_tokens - 1) / s.tile_tokens;
}

__device__ __forceinline__ int row_groups_of(const SharedArgs& s, int rows) {
    return (int)(((long long)rows * s.a.group + kPrefillRows - 1) / kPrefillRows);
}

// A unit of T tiles at `at` on the line whose shares are `share` long: workgroups first .. last hold a piece
// of it, and cut(w) is the tile where the piece of workgroup w + 1 begins. Cuts near an end are moved to it, so that
// no piece is a few tiles; the pieces that are left follow each other (a share is longer than what two cuts are moved).
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
        const int k = (w + 1) * share - at - kSharedUnitCost;
        return k < kSharedLeastPart ? 0 : k > T - kSharedLeastPart ? T : k;
    }
    __device__ int first_piece() const { return first + (first < last && cut(first) == 0); }
    __device__ int pieces() const { return last - (first < last && cut(last - 1) == T) + 1 - first_piece(); }
    // Whether the line's share w begins, or ends, in the unit.
    __device__ bool begins(int w) const { return w * share >= at; }
    __device__ bool ends(int w, int line) const { return w < last || (w + 1) * share == end() || end() == line; }
};

// Inclusive sum over the workgroup's N threads, and the total. `part` holds a value per wave.
template <int N>
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
#pragma unroll
    for (int w = 0; w < N / 64; ++w) {
        before += w < wave ? part[w] : 0;
        total += part[w];
    }
    return before + x;
}

// One workgroup of N threads lists the work. A thread has sequence b = thread (and b + N, ..), and group g = thread;
// records are in LDS for batches of up to N sequences and N groups, in scratch otherwise.
template <int N>
__global__ __launch_bounds__(N) void attn_shared_plan_kernel(SharedArgs s) {
    const AttnArgs& a = s.a;
    __shared__ int64_t part[N / 64], red_sum[N / 64];
    __shared__ int bad_groups;
    __shared__ int l_starts[N + 1];
    __shared__ int4 l_seqs[N], l_groups[N];
    __shared__ int2 l_counts[N];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const bool few = s.G <= N;
    int4* seqs = a.B <= N ? l_seqs : s.seqs;
    int4* groups = few ? l_groups : s.groups;
    int2* counts = few ? l_counts : s.counts;
    const int32_t* starts = few ? l_starts : s.group_starts;
    if (t == 0) bad_groups = 0;
    // Sequences: {first row, rows, context length, -1}, no rows where something is wrong.
    for (int b = t; b < a.B; b += N) {
        const int64_t c = a.ctx_lens[b];
        const int q0 = a.q_start ? a.q_start[b] : b, q1 = a.q_start ? a.q_start[b + 1] : b + 1;
        int err = 0;
        if (c < 0 || c > (int64_t)a.max_blocks * a.bs) err |= ERR_CTX_LEN;
        if (q0 < 0 || q1 < q0 || q1 > a.total_q || q1 - q0 > a.max_q_len) err |= ERR_Q_LAYOUT;
        if (err) latch_error(a.err, err);
        seqs[b] = make_int4(q0, err ? 0 : q1 - q0, err ? 0 : (int)c, -1);
    }
    __syncthreads();
    // Groups: {first row, rows, common tiles, first unit}.
    for (int g = t; g < s.G; g += N) {
        const int s0 = s.group_starts[g], s1 = s.group_starts[g + 1], nb = s.group_blocks[g];
        if (few) {
            l_starts[g] = s0;
            if (g == s.G - 1) l_starts[s.G] = s1;
        }
        int4 e = make_int4(0, 0, 0, 0);
        if (s0 < 0 || s1 < s0 || s1 > a.B) {
            bad_groups = 1;
        } else if (nb < 0 || nb > a.max_blocks) {
            latch_error(a.err, ERR_GROUPS);
        } else if (nb > 0) {
            const int q0 = a.q_start ? a.q_start[s0] : s0, q1 = a.q_start ? a.q_start[s1] : s1;
            if (q0 >= 0 && q0 <= q1 && q1 <= a.total_q)
                e = make_int4(q0, q1 - q0, (int)((long long)nb * a.bs / s.tile_tokens), 0);
        }
        groups[g] = e;
        counts[g] = make_int2(0, 0);
    }
    __syncthreads();
    const int G = bad_groups ? 0 : s.G;
    if (bad_groups && t == 0) latch_error(a.err, ERR_GROUPS);
    // The group that a sequence shares with, if every row of it sees the common tokens.
    for (int b = t; b < a.B; b += N) {
        const int4 e = seqs[b];
        if (e.y == 0 || G == 0) continue;
        int lo = 0, hi = G;  // the last group that starts at or before b is lo - 1
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (starts[mid] <= b) lo = mid + 1;
            else hi = mid;
        }
        const int g = lo - 1;
        if (g < 0 || b >= starts[g + 1]) continue;
        const int4 gr = groups[g];
        const long long sees = a.causal ? (long long)e.z - e.y + 1 : e.z;
        if (gr.z > 0 && sees >= (long long)gr.z * s.tile_tokens && e.x >= gr.x && e.x + e.y <= gr.x + gr.y) {
            seqs[b].w = g;
            atomicAdd(&counts[g].x, 1);
            atomicAdd(&counts[g].y, row_groups_of(s, e.y));
        }
    }
    __syncthreads();
    // A group shares where that saves workgroups tiles. The common units' places: {length, units} summed over the groups.
    int64_t line = 0, units = 0;
    for (int g0 = 0; g0 < G; g0 += N) {
        const int g = g0 + t;
        int64_t len = 0, n = 0;
        if (g < G) {
            const int4 gr = groups[g];
            const int2 k = counts[g];
            const int rgs = row_groups_of(s, gr.y);
            if (k.x < 2 || (long long)(k.y - rgs) * gr.z < 1) {
                groups[g].z = 0;
            } else {
                n = rgs;
                len = n * (gr.z + kSharedUnitCost);
            }
        }
        int64_t all_len, all_n;
        const int64_t at = line + block_scan<N>(len, part, all_len) - len, u = units + block_scan<N>(n, part, all_n) - n;
        if (g < G) groups[g].w = (int)min(u, (int64_t)INT32_MAX), counts[g] = make_int2((int)at, 0);
        line += all_len;
        units += all_n;
    }
    __syncthreads();
    const int64_t common_units = units, common_line = line;
    auto common_tiles = [&](const int4& e) -> int { return e.w >= 0 ? groups[e.w].z : 0; };
    // The whole line: with the sequences' own units.
    int64_t sum = 0;
    for (int b = t; b < a.B; b += N) {
        const int4 e = seqs[b];
        const int first = common_tiles(e), nrg = row_groups_of(s, e.y);
        for (int rg = 0; rg < nrg; ++rg) sum += visible_tiles(s, rg, e.y, e.z) - first + kSharedUnitCost;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (lane == 0) red_sum[wave] = sum;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < N / 64; ++w) line += red_sum[w];
    const int whole = (int)line;  // in 31 bits, as the host has bounded it, unless rows overlap
    const int share = (int)max((line + s.lanes - 1) / s.lanes, (int64_t)kSharedLeastShare);
    // Rows that overlap around an invalid range can make more units than were sized: latch it and run nothing.
    bool over = common_units > s.common_cap || line > INT32_MAX - share;
    for (int g = wave; g < G && !over; g += N / 64) {
        const int4 gr = groups[g];
        if (gr.z == 0) continue;
        const int at = counts[g].x;
        const int len = gr.z + kSharedUnitCost, rgs = row_groups_of(s, gr.y), b0 = starts[g];
        const int most = (len - 1) / share + 2;  // pieces of a unit at most
        for (int x = lane; x < rgs * most; x += 64) {
            const int r = x / most, u = gr.w + r;
            const Pieces p(at + r * len, gr.z, share);
            const int w = p.first + (x - r * most);
            if (x == r * most) s.common_parts[u] = make_int2(u + p.first_piece(), p.pieces());
            if (w > p.last) continue;
            const int from = p.cut(w - 1), to = p.cut(w);
            s.list[2 * (u + w)] = make_int4(from < to ? b0 : -1, gr.x, gr.y, gr.z * s.tile_tokens);
            s.list[2 * (u + w) + 1] = make_int4(r * kPrefillRows, from, (to - from) | kSharedAll, u + w);
            if (p.begins(w)) s.ranges[w].x = u;
            if (p.ends(w, whole)) s.ranges[w].y = u;
        }
    }
    // The sequences' own units, and the row groups to merge.
    int64_t merges = 0;
    line = common_line;
    for (int b0 = 0; b0 < a.B; b0 += N) {
        const int b = b0 + t;
        int4 e = make_int4(0, 0, 0, -1);
        int first = 0, nrg = 0;
        int64_t len = 0;
        if (b < a.B) {
            e = seqs[b];
            first = common_tiles(e);
            nrg = row_groups_of(s, e.y);
            for (int rg = 0; rg < nrg; ++rg) len += visible_tiles(s, rg, e.y, e.z) - first + kSharedUnitCost;
        }
        int64_t all_len, all_n;
        int64_t at = line + block_scan<N>(len, part, all_len) - len, u = units + block_scan<N>(nrg, part, all_n) - nrg;
        line += all_len;
        units += all_n;
        over = over || units - common_units > s.own_cap;
        // Merges: counted first, as the pieces of a unit decide.
        int64_t mine = 0;
        if (!over) {
            int p0 = (int)at;
            for (int rg = 0; rg < nrg; ++rg) {
                const Pieces p(p0, visible_tiles(s, rg, e.y, e.z) - first, share);
                mine += first > 0 || p.pieces() > 1;
                p0 = p.end();
            }
        }
        int64_t all_merges;
        int64_t merge = merges + block_scan<N>(mine, part, all_merges) - mine;
        merges += all_merges;
        if (over) continue;
        const int4 gr = first > 0 ? groups[e.w] : make_int4(0, 0, 0, -1);
        for (int rg = 0; rg < nrg; ++rg, ++u) {
            const Pieces p((int)at, visible_tiles(s, rg, e.y, e.z) - first, share);
            at = p.end();
            const int pieces = p.pieces();
            const bool parked = first > 0 || pieces > 1, none = first > 0 && p.T == 0;
            for (int w = p.first; w <= p.last; ++w) {
                const int from = p.cut(w - 1), to = p.cut(w);
                const bool piece = !none && (from < to || (p.T == 0 && w == p.last));
                s.list[2 * (u + w)] = make_int4(piece ? b : -1, e.x, e.y, e.z);
                s.list[2 * (u + w) + 1] = make_int4(rg * kPrefillRows, first + from, to - from, parked ? (int)(u - common_units) + w : -1);
                if (p.begins(w)) s.ranges[w].x = (int)u;
                if (p.ends(w, whole)) s.ranges[w].y = (int)u;
            }
            if (parked) {
                s.merges[2 * merge] = make_int4(e.x, e.y, rg * kPrefillRows, (e.x - gr.x) * a.group + rg * kPrefillRows);
                s.merges[2 * merge + 1] = make_int4((int)(u - common_units) + p.first_piece(), none ? 0 : pieces, gr.w, 0);
                ++merge;
            }
        }
    }
    if (t == 0) {
        if (over) latch_error(a.err, ERR_PLAN);
        s.head[0] = over ? 0 : (whole + share - 1) / share;
        s.head[1] = over ? 0 : (int)merges;
    }
}

// Merges the partial states of the listed row groups. A workgroup takes a slice of one row group's (row, four
// columns) for one kv head, rows fastest, so that the lanes read the neighbouring rows that a state keeps together.
template <int DR>
__global__ __launch_bounds__(kThreads) void attn_shared_combine_kernel(SharedArgs s) {
    const AttnArgs& a = s.a;
    constexpr int DT = (DR + 31) / 32, Q = DR / 4;
    const int entry = (int)blockIdx.x / a.Hkv, kvh = (int)blockIdx.x - entry * a.Hkv;
    if (entry >= s.head[1]) return;
    const int4 e = s.merges[2 * entry], f = s.merges[2 * entry + 1];
    const int rows = min(kPrefillRows, e.y * a.group - e.z);
    const int x = (int)blockIdx.y * kThreads + threadIdx.x;
    if (x >= rows * Q) return;
    const int c = x / rows, r = x - c * rows;  // columns 4 c .. 4 c + 3 of row e.z + r
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
    constexpr int kBatch = 8;  // loads in flight; an index past the last reads the last one again with weight 0
    for (int i0 = 0; i0 < n; i0 += kBatch) {
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
    const float inv = L > 0.f ? 1.f / L : 0.f;
    SeqInfo si;
    si.q0 = e.x;
    si.kvh = kvh;
    store_row4<DR>(a, out_row(a, si, e.z + r), 4 * c, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

template <int DR>
void launch_combine(const SharedArgs& s, hipStream_t stream) {
    const AttnArgs& a = s.a;
    const int rows = a.rows_cap < kPrefillRows ? a.rows_cap : kPrefillRows;
    attn_shared_combine_kernel<DR><<<dim3((unsigned)((long long)s.own_cap * a.Hkv), (unsigned)((rows * (DR / 4) + kThreads - 1) / kThreads)),
                                     kThreads, 0, stream>>>(s);
}

}  // namespace

hipError_t launch_shared_bf16(const SharedArgs& s, hipStream_t stream);
hipError_t launch_shared_wide(const SharedArgs& s, hipStream_t stream);
hipError_t launch_shared_f32(const SharedArgs& s, hipStream_t stream);

hipError_t launch_attention_shared(const SharedArgs& s, hipStream_t stream) {
    const AttnArgs& a = s.a;
    if (a.B <= 256 && s.G <= 256) attn_shared_plan_kernel<256><<<dim3(1), 256, 0, stream>>>(s);
    else attn_shared_plan_kernel<1024><<<dim3(1), 1024, 0, stream>>>(s);
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
