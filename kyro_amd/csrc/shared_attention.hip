// Paged attention for a batch whose sequences share prefixes (block tables that start with the same blocks).
//
// A softmax over a context is the merge of softmaxes over its parts, so the tokens that a group of sequences has in
// common need not be walked once a sequence: all rows of the group, which are consecutive rows of the query, see all
// of them, and become the rows of one product. What remains of each sequence, its own tokens, is walked as before.
//   * attn_shared_plan_kernel: one workgroup checks the groups, decides for each whether its common tokens are worth
//     a pass of their own, and lists the work: row groups of 128 rows over common tokens, and each sequence's
//     row groups over its own, in parts of at most a workgroup's share of all, longest first.
//   * attn_prefill_kernel<.., SHARED> (prefill_attention.hip) runs the list; products of common tokens and streams
//     of own ones share the chip.
//   * attn_shared_combine_kernel merges each row's partial states, common ones and own ones.
// Common tokens are taken in whole tiles (64 tokens, 32 in f32 and above head dim 128), so that no tile needs a
// mask at its start; what is left of the last one counts as each sequence's own.
#include "attention_rows.hpp"
#include "common.hpp"
#include "kernels.hpp"

namespace kyro {

namespace {

constexpr int kThreads = 256;
constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;

// Tiles up to the last token that row group rg of q_len rows sees, or -1 where it has no rows.
__device__ __forceinline__ int visible_tiles(const PrefillArgs& p, int rg, int q_len, int ctx) {
    const int rows = q_len * p.a.group;
    if (rg * kPrefillRows >= rows) return -1;
    const int last = min((rg + 1) * kPrefillRows, rows) - 1;
    const int vis = p.a.causal ? ctx - q_len + last / p.a.group + 1 : ctx;
    return (max(vis, 0) + p.tile_tokens - 1) / p.tile_tokens;
}

__device__ __forceinline__ int row_groups_of(const PrefillArgs& p, int rows) {
    return (int)(((long long)rows * p.a.group + kPrefillRows - 1) / kPrefillRows);
}

__global__ __launch_bounds__(kPlanThreads) void attn_shared_plan_kernel(SharedArgs s) {
    const PrefillArgs& p = s.f;
    const AttnArgs& a = p.a;
    constexpr int kBuckets = kPlanThreads;
    __shared__ int bucket[kBuckets];
    __shared__ long long red_sum[kPlanWaves];
    __shared__ int red_max[kPlanWaves], wave_tot[kPlanWaves];
    __shared__ int n_common, n_tail, n_comb, bad_groups;
    __shared__ int4 l_seqs[kPlanThreads], l_groups[kPlanThreads];
    __shared__ int2 l_counts[kPlanThreads];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    int4* seqs = a.B <= kPlanThreads ? l_seqs : s.seqs;
    int4* groups = s.G <= kPlanThreads ? l_groups : s.groups;
    int2* counts = s.G <= kPlanThreads ? l_counts : s.counts;
    bucket[t] = 0;
    if (t == 0) n_common = n_tail = n_comb = bad_groups = 0;
    __syncthreads();
    // Groups: their rows and common tiles.
    for (int g = t; g < s.G; g += kPlanThreads) {
        const int s0 = s.group_starts[g], s1 = s.group_starts[g + 1], nb = s.group_blocks[g];
        int4 e = make_int4(0, 0, 0, 0);
        if (s0 < 0 || s1 < s0 || s1 > a.B) {
            bad_groups = 1;
        } else if (nb < 0 || nb > a.max_blocks) {
            latch_error(a.err, ERR_GROUPS);
        } else {
            const int q0 = a.q_start ? a.q_start[s0] : s0, q1 = a.q_start ? a.q_start[s1] : s1;
            if (q0 >= 0 && q0 <= q1 && q1 <= a.total_q)
                e = make_int4(q0, q1 - q0, (int)((long long)nb * a.bs / p.tile_tokens), 0);
        }
        groups[g] = e;
        counts[g] = make_int2(0, 0);
    }
    __syncthreads();
    const int G = bad_groups ? 0 : s.G;
    if (bad_groups && t == 0) latch_error(a.err, ERR_GROUPS);
    // Sequences: the group each shares with, if every row of it sees the common tokens.
    for (int b = t; b < a.B; b += kPlanThreads) {
        const int64_t c = a.ctx_lens[b];
        const int q0 = a.q_start ? a.q_start[b] : b, q1 = a.q_start ? a.q_start[b + 1] : b + 1;
        int err = 0;
        if (c < 0 || c > (int64_t)a.max_blocks * a.bs) err |= ERR_CTX_LEN;
        if (q0 < 0 || q1 < q0 || q1 > a.total_q || q1 - q0 > a.max_q_len) err |= ERR_Q_LAYOUT;
        if (err) latch_error(a.err, err);
        int4 e = make_int4(q0, err ? 0 : q1 - q0, err ? 0 : (int)c, -1);
        if (G > 0 && e.y > 0) {
            int lo = 0, hi = G;  // the last group that starts at or before b
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (s.group_starts[mid] <= b) lo = mid + 1;
                else hi = mid;
            }
            const int g = lo - 1;
            if (g >= 0 && b < s.group_starts[g + 1]) {
                const int4 gr = groups[g];
                const long long sees = a.causal ? (long long)e.z - e.y + 1 : e.z;
                if (gr.z > 0 && sees >= (long long)gr.z * p.tile_tokens && e.x >= gr.x && e.x + e.y <= gr.x + gr.y) {
                    e.w = g;
                    atomicAdd(&counts[g].x, 1);
                    atomicAdd(&counts[g].y, row_groups_of(p, e.y));
                }
            }
        }
        seqs[b] = e;
    }
    __syncthreads();
    // A group shares where that saves workgroups their tiles.
    for (int g = t; g < G; g += kPlanThreads) {
        const int2 n = counts[g];
        if (n.x < 2 || (long long)(n.y - row_groups_of(p, groups[g].y)) * groups[g].z < 1) groups[g].z = 0;
    }
    __syncthreads();
    auto shared_tiles = [&](const int4& e) -> int { return e.w >= 0 ? groups[e.w].z : 0; };
    // The work in tiles, and the longest piece.
    const unsigned flat = (unsigned)a.B * (unsigned)a.row_groups;  // below 2^31 (the host checks)
    auto own_tiles = [&](unsigned f, int& b, int& rg, int4& e, int& first) -> int {
        b = (int)(f / (unsigned)a.row_groups);
        rg = (int)(f - (unsigned)b * (unsigned)a.row_groups);
        e = seqs[b];
        first = shared_tiles(e);
        const int T = visible_tiles(p, rg, e.y, e.z);
        return T < 0 ? -1 : T - first;
    };
    long long sum = 0;
    int mx = 0;
    int b, rg, first;
    int4 e;
    for (unsigned f = t; f < flat; f += kPlanThreads) {
        const int T = own_tiles(f, b, rg, e, first);
        sum += max(T, 0);
        mx = max(mx, T);
    }
    for (int g = t; g < G; g += kPlanThreads) {
        const int T = groups[g].z;
        if (T == 0) continue;
        sum += (long long)row_groups_of(p, groups[g].y) * T;
        mx = max(mx, T);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        sum += __shfl_xor(sum, o, 64);
        mx = max(mx, __shfl_xor(mx, o, 64));
    }
    if (lane == 0) {
        red_sum[wave] = sum;
        red_max[wave] = mx;
    }
    __syncthreads();
    sum = 0;
    mx = 0;
    for (int w = 0; w < kPlanWaves; ++w) {
        sum += red_sum[w];
        mx = max(mx, red_max[w]);
    }
    const long long share = (sum * a.Hkv + p.slots - 1) / p.slots + p.split_cost;
    const int C = (int)min((long long)max(mx, 1), share);
    auto split = [&](int T, int& len, int& np) {
        len = T;
        np = 1;
        if (T > C) {
            np = (T + C - 1) / C;
            len = (T + np - 1) / np;
            np = (T + len - 1) / len;
        }
    };
    int shift = 0;
    while ((C >> shift) >= kBuckets) ++shift;
    auto bucket_of = [&](int len) { return (C - len) >> shift; };
    // Twice over the work: entries of each length, then (their places known) the entries.
    for (int pass = 0; pass < 2; ++pass) {
        for (unsigned f = t; f < flat; f += kPlanThreads) {
            const int T = own_tiles(f, b, rg, e, first);
            if (T < 0 || (T == 0 && first > 0)) continue;
            int len, np;
            split(T, len, np);
            if (pass == 0) {
                if (np > 1) atomicAdd(&bucket[bucket_of(len)], np - 1);
                atomicAdd(&bucket[bucket_of(T - (np - 1) * len)], 1);
                continue;
            }
            const bool parked = np > 1 || first > 0;
            int base = -1;
            if (parked) {
                const int part = atomicAdd(&n_tail, np);
                base = part + np <= s.tail_cap ? (s.common_cap * 4 + part * p.tail_waves) * a.Hkv : 0;
            }
            for (int i = 0; i < np; ++i) {
                const int nt = i + 1 < np ? len : T - (np - 1) * len;
                const int pos = atomicAdd(&bucket[bucket_of(nt)], 1);
                if (pos < p.list_cap) {
                    p.list[2 * pos] = make_int4(b, e.x, e.y, e.z);
                    p.list[2 * pos + 1] = make_int4(rg * kPrefillRows, first + i * len, nt,
                                                    parked ? base + i * p.tail_waves * a.Hkv : -1);
                }
            }
            if (np > 1 && first == 0) {
                const int x = atomicAdd(&n_comb, 1);
                if (x < s.comb_cap) {
                    p.comb[2 * x] = make_int4(e.x, e.y, rg * kPrefillRows, 0);
                    p.comb[2 * x + 1] = make_int4(base, np, 0, 0);
                }
            } else if (first > 0) {
                const int x = atomicAdd(&n_comb, 1);
                if (x < s.comb_cap) {
                    p.comb[2 * x] = make_int4(e.x, e.y, rg * kPrefillRows, e.w);
                    p.comb[2 * x + 1] = make_int4(base, np, -1, 0);
                }
            }
        }
        // Row groups that see common tokens alone.
        if (pass == 1)
            for (unsigned f = t; f < flat; f += kPlanThreads) {
                const int T = own_tiles(f, b, rg, e, first);
                if (T != 0 || first == 0) continue;
                const int x = atomicAdd(&n_comb, 1);
                if (x < s.comb_cap) {
                    p.comb[2 * x] = make_int4(e.x, e.y, rg * kPrefillRows, e.w);
                    p.comb[2 * x + 1] = make_int4(0, 0, -1, 0);
                }
            }
        for (int g = wave; g < G; g += kPlanWaves) {
            const int4 gr = groups[g];
            if (gr.z == 0) continue;
            int len, np;
            split(gr.z, len, np);
            const int nrg = row_groups_of(p, gr.y);
            int part0 = 0;
            if (pass == 1) {
                if (lane == 0) part0 = atomicAdd(&n_common, nrg * np);
                part0 = __builtin_amdgcn_readfirstlane(part0);
                if (lane == 0) groups[g].w = part0;
            }
            const bool fits = part0 + nrg * np <= s.common_cap;
            const int b0 = s.group_starts[g];
            for (int x = lane; x < nrg * np; x += 64) {  // the row groups of one part next to each other
                const int i = x / nrg, r = x - i * nrg;
                const int nt = i + 1 < np ? len : gr.z - (np - 1) * len;
                const int pos = atomicAdd(&bucket[bucket_of(nt)], 1);
                if (pass == 1 && pos < p.list_cap) {
                    p.list[2 * pos] = make_int4(b0, gr.x, gr.y, gr.z * p.tile_tokens);
                    p.list[2 * pos + 1] = make_int4(r * kPrefillRows, i * len, nt | kSharedAll,
                                                    fits ? (part0 + r * np + i) * 4 * a.Hkv : 0);
                }
            }
        }
        __syncthreads();
        if (pass == 0) {
            const int mine = bucket[t];
            const int incl = wave_incl_scan_i(mine);
            if (lane == 63) wave_tot[wave] = incl;
            __syncthreads();
            int before = 0, total = 0;
            for (int w = 0; w < kPlanWaves; ++w) {
                before += w < wave ? wave_tot[w] : 0;
                total += wave_tot[w];
            }
            bucket[t] = before + incl - mine;
            if (t == 0) red_max[0] = total;
            __syncthreads();
        }
    }
    const int total = red_max[0];
    // More entries or parts than were sized (rows that overlap around an invalid range): latch it and run nothing.
    const bool over = total > p.list_cap || n_common > s.common_cap || n_tail > s.tail_cap || n_comb > s.comb_cap;
    for (int x = t; x < min(n_comb, s.comb_cap); x += kPlanThreads) {
        if (p.comb[2 * x + 1].z != -1) continue;
        const int4 u = p.comb[2 * x], v = p.comb[2 * x + 1];
        const int4 gr = groups[u.w];
        int len, np;
        split(gr.z, len, np);
        p.comb[2 * x] = make_int4(u.x, u.y, u.z, (u.x - gr.x) * a.group + u.z);
        p.comb[2 * x + 1] = make_int4(v.x, v.y, gr.w * 4 * a.Hkv, np);
    }
    if (t == 0) {
        if (over) latch_error(a.err, ERR_PLAN);
        p.head[0] = over ? 0 : total;
        p.head[1] = over ? 0 : n_comb;
    }
}

// Merges the partial states of the listed row groups. A workgroup takes a slice of one row group's (row, four
// columns) for one kv head, rows fastest, so that the lanes read the neighbouring rows that a state keeps together.
template <int DR>
__global__ __launch_bounds__(kThreads) void attn_shared_combine_kernel(SharedArgs s) {
    const PrefillArgs& p = s.f;
    const AttnArgs& a = p.a;
    constexpr int DT = (DR + 31) / 32, Q = DR / 4;
    const int entry = (int)blockIdx.x / a.Hkv, kvh = (int)blockIdx.x - entry * a.Hkv;
    if (entry >= p.head[1]) return;
    const int4 e = p.comb[2 * entry], f = p.comb[2 * entry + 1];
    const int rows = min(kPrefillRows, e.y * a.group - e.z);
    const int x = (int)blockIdx.y * kThreads + threadIdx.x;
    if (x >= rows * Q) return;
    const int c = x / rows, r = x - c * rows;  // columns 4 c .. 4 c + 3 of row e.z + r
    const int dt = c / 8, k = c / 2 % 4, h = c % 2;
    float M = kNegInf, L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    auto merge = [&](size_t wv0, size_t step, int n, int row) {
        const int col = row & 31;
        const size_t at = wv0 + (row >> 5);
        constexpr int kBatch = 8;  // loads in flight; an index past the last reads the last one again with weight 0
        for (int i0 = 0; i0 < n; i0 += kBatch) {
            float m[kBatch], l[kBatch];
            float4 v[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const size_t wv = at + (size_t)min(i0 + i, n - 1) * step;
                m[i] = a.ws_m[wv * 32 + col];
                l[i] = a.ws_l[wv * 32 + col];
                v[i] = reinterpret_cast<const float4*>(a.ws_acc)[((wv * DT + dt) * 4 + k) * 64 + 32 * h + col];
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
    };
    // A common part: its row group's 4 wave slots for each kv head; the row groups' parts follow each other.
    const int g = e.w + r;
    if (f.w > 0)
        merge((size_t)f.z + ((size_t)(g / kPrefillRows) * f.w * a.Hkv + kvh) * 4, (size_t)a.Hkv * 4, f.w, g % kPrefillRows);
    merge((size_t)f.x + (size_t)kvh * p.tail_waves, (size_t)a.Hkv * p.tail_waves, f.y, r);
    const float inv = L > 0.f ? 1.f / L : 0.f;
    SeqInfo si;
    si.q0 = e.x;
    si.kvh = kvh;
    store_row4<DR>(a, out_row(a, si, e.z + r), 4 * c, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

template <int DR>
void launch_combine(const SharedArgs& s, hipStream_t stream) {
    const AttnArgs& a = s.f.a;
    const int rows = a.rows_cap < kPrefillRows ? a.rows_cap : kPrefillRows;
    attn_shared_combine_kernel<DR><<<dim3((unsigned)((long long)s.comb_cap * a.Hkv), (unsigned)((rows * (DR / 4) + kThreads - 1) / kThreads)),
                                     kThreads, 0, stream>>>(s);
}

}  // namespace

hipError_t launch_shared_bf16(const PrefillArgs& p, hipStream_t stream);
hipError_t launch_shared_wide(const PrefillArgs& p, hipStream_t stream);
hipError_t launch_shared_f32(const PrefillArgs& p, hipStream_t stream);

hipError_t launch_attention_shared(const SharedArgs& s, hipStream_t stream) {
    const AttnArgs& a = s.f.a;
    attn_shared_plan_kernel<<<dim3(1), kPlanThreads, 0, stream>>>(s);
    const hipError_t e = !a.dtype_bf16 ? launch_shared_f32(s.f, stream) : a.D > 128 ? launch_shared_wide(s.f, stream) : launch_shared_bf16(s.f, stream);
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
