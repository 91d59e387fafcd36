// Eviction from a paged cache by accumulated attention weight (gfx950).
//
// For each (sequence, kv head) with n > budget tokens: key(t) = the weight's bits mapped so that unsigned
// order is the weights' order (protected tokens above all, NaN with -infinity at the bottom); the budget-th
// largest key T by radix selection; tokens above T stay, and of those equal to T the lowest slots fill
// the rest. A slot < budget whose token goes (a hole) takes the token of a kept slot >= budget (a mover),
// both in ascending order. Holes and movers are as many, and no mover's slot is written, so the moves need
// no order among themselves and what is moved is only what has to be: a budget of 2048 with 256 tokens over
// it moves at most 256 of them, where closing the gaps in order would move most of 2048.
//
// evict_select_kernel: one workgroup a (sequence, kv head). Selection reads 8 bytes a token once; the keys
// stay in LDS (up to kLdsKeys of them) for the three passes over 11, 11 and 10 bits. The first digit holds
// the sign, the exponent and two bits of the mantissa, so weights that fall over many octaves spread over
// its bins. Lists of holes and movers go to scratch. evict_move_kernel: copies K and V rows, 16 bytes a lane.
// What bounds the pair: latency of the passes for few tokens, HBM for many.
#include "common.hpp"
#include "kernels.hpp"

namespace kyro {
namespace {

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kBins = 2048;
constexpr int kMoveThreads = 256;

// Order-preserving bits: a < b as floats <=> rank(a) < rank(b); -0 ranks as +0, NaN as -infinity.
__device__ __forceinline__ uint32_t rank_bits(float w) {
    uint32_t u = __float_as_uint(w);
    if ((u & 0x7fffffffu) > 0x7f800000u) u = 0xff800000u;
    if (u == 0x80000000u) u = 0;
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Maximum over the workgroup; every thread gets it. red: one int per wave.
__device__ __forceinline__ int block_max(int v, int* red) {
    for (int m = 32; m; m >>= 1) v = max(v, __shfl_xor(v, m, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
    for (int i = 1; i < kSelWaves; ++i) v = max(v, red[i]);
    __syncthreads();
    return v;
}

// Is the sequence to be worked on? Latches what is wrong with it. Uniform over the workgroup.
__device__ bool evict_valid(const EvictArgs& a, int b, int64_t n, int64_t* row, int* bad_any) {
    int bad = 0;
    *row = b;
    if (a.state_rows) {
        const int r = a.state_rows[b];
        *row = r;
        if (r < 0 || r >= a.num_state_rows) bad = ERR_STATE_ROW;
        for (int i = threadIdx.x; i < a.B; i += blockDim.x)
            if (i != b && a.state_rows[i] == r) bad = ERR_STATE_ROW;
    }
    if (n < 0 || n > a.cap) {
        bad |= ERR_CTX_LEN;
    } else {
        const int64_t blocks = (n + a.bs - 1) / a.bs;
        for (int64_t i = threadIdx.x; i < blocks; i += blockDim.x) {
            const int64_t id = a.table[(size_t)b * a.max_blocks + i];
            if (id < 0 || id >= a.num_blocks) bad |= ERR_BLOCK_ID;
        }
    }
    if (bad) atomicOr(bad_any, bad);  // LDS
    __syncthreads();
    const int all = *bad_any;
    if (all && threadIdx.x == 0) latch_error(a.err, all);
    return all == 0;
}

// The bin that holds the `want`-th largest of the histogram (want >= 1), and how many are in the bins
// above it. One wave scans; every thread gets the answer through out[2].
__device__ __forceinline__ void find_bin(const int* hist, int want, int* out) {
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x;
        constexpr int per = kBins / 64;
        // Lane 0 holds the largest bins.
        int mine = 0;
        for (int i = 0; i < per; ++i) mine += hist[kBins - 1 - lane * per - i];
        const int incl = wave_incl_scan_i(mine);
        const unsigned long long reach = __ballot(incl >= want);
        const int first = __ffsll((unsigned long long)reach) - 1;
        if (lane == first) {
            int above = incl - mine, bin = kBins - 1 - lane * per;
            while (above + hist[bin] < want) above += hist[bin--];
            out[0] = bin;
            out[1] = above;
        }
    }
    __syncthreads();
}

__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(EvictArgs a) {
    extern __shared__ uint32_t lds_keys[];  // a.lds_keys entries
    __shared__ int hist[kBins];
    __shared__ int red[3 * kSelWaves];
    __shared__ int found[2];
    __shared__ int bad_any;
    const int b = blockIdx.x / a.Hkv, h = blockIdx.x % a.Hkv;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t n64 = a.ctx_lens[b];
    if (tid == 0) bad_any = 0;
    __syncthreads();
    int64_t row;
    const bool ok = evict_valid(a, b, n64, &row, &bad_any);
    if (tid == 0) {
        a.num_moves[blockIdx.x] = 0;
        if (h == 0) a.out_ctx_lens[b] = ok && n64 > a.budget ? a.budget : n64;
    }
    if (!ok) return;
    const int n = (int)n64, budget = a.budget;
    const size_t base = ((size_t)row * a.Hkv + h) * a.max_tokens;
    const float* w = a.weights + base;
    const int32_t* pos = a.positions + base;
    float* ow = a.out_weights + base;
    int32_t* op = a.out_positions + base;
    const bool copy = ow != w, copy_pos = op != pos;
    if (n <= budget) {
        for (int t = tid; t < n; t += kSelThreads) {
            if (copy) ow[t] = w[t];
            if (copy_pos) op[t] = pos[t];
        }
        return;
    }

    int newest = INT32_MIN;
    for (int t = tid; t < n; t += kSelThreads) newest = max(newest, pos[t]);
    newest = block_max(newest, red);
    const int64_t from = (int64_t)newest - a.recent;  // positions above it are protected
    const bool in_lds = n <= a.lds_keys;
    const auto key_of = [&](int t) -> uint32_t {
        const int p = pos[t];
        return p < a.sink || (int64_t)p > from ? 0xffffffffu : rank_bits(w[t]);
    };

    // The budget-th largest key, digit by digit from the top; `want` counts within the keys that share the
    // digits found so far.
    uint32_t prefix = 0;
    int want = budget;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t mask = pass == 2 ? 1023u : 2047u;
        for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
        __syncthreads();
        for (int t = tid; t < n; t += kSelThreads) {
            uint32_t k;
            if (pass == 0 || !in_lds) {
                k = key_of(t);
                if (in_lds) lds_keys[t] = k;
            } else {
                k = lds_keys[t];
            }
            const bool same = pass == 0 || (k >> (pass == 1 ? 21 : 10)) == prefix;
            if (same) atomicAdd(&hist[(k >> shift) & mask], 1);
        }
        __syncthreads();
        find_bin(hist, want, found);
        prefix = (prefix << (pass == 2 ? 10 : 11)) | (uint32_t)found[0];
        want -= found[1];
        __syncthreads();
    }
    const uint32_t T = prefix;  // `want` of the keys equal to T stay, those of the lowest slots

    // Slot order from here on: wave i owns slots [i seg, (i + 1) seg). Equal keys before each wave's first.
    const int seg = ((n + kSelThreads - 1) / kSelThreads) * 64;
    const int t0 = min(n, wave * seg), t1 = min(n, t0 + seg);
    int eq = 0;
    for (int t = t0; t < t1; t += 64) {
        const int at = t + lane;
        const uint32_t k = at < t1 ? (in_lds ? lds_keys[at] : key_of(at)) : 0u;
        eq += __popcll(__ballot(at < t1 && k == T));
    }
    if (lane == 0) red[wave] = eq;
    __syncthreads();
    int eq_before = 0;
    for (int i = 0; i < wave; ++i) eq_before += red[i];
    // Twice over the wave's slots: holes and movers counted, then listed behind those of the waves before.
    const unsigned long long below = lane == 0 ? 0ull : (~0ull >> (64 - lane));
    int holes = 0, movers = 0, hole_at = 0, mover_at = 0;
    int32_t* hole_list = a.moves + (size_t)blockIdx.x * 2 * a.max_moves;
    int32_t* mover_list = hole_list + a.max_moves;
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
        int seen = eq_before;
        for (int t = t0; t < t1; t += 64) {
            const int at = t + lane;
            const bool in = at < t1;
            const uint32_t k = in ? (in_lds ? lds_keys[at] : key_of(at)) : 0u;
            const unsigned long long ties = __ballot(in && k == T);
            const bool keep = in && (k > T || (k == T && seen + __popcll(ties & below) < want));
            seen += __popcll(ties);
            const unsigned long long hb = __ballot(in && !keep && at < budget), mb = __ballot(keep && at >= budget);
            if (pass == 0) {
                holes += __popcll(hb);
                movers += __popcll(mb);
            } else {
                if (in && !keep && at < budget) hole_list[hole_at + __popcll(hb & below)] = at;
                if (keep && at >= budget) mover_list[mover_at + __popcll(mb & below)] = at;
                hole_at += __popcll(hb);
                mover_at += __popcll(mb);
                if (keep && at < budget) {
                    if (copy) ow[at] = w[at];
                    if (copy_pos) op[at] = pos[at];
                }
            }
        }
        if (pass == 0) {
            __syncthreads();  // red's tie counts have been read
            if (lane == 0) {
                red[kSelWaves + wave] = holes;
                red[2 * kSelWaves + wave] = movers;
            }
            __syncthreads();
            for (int i = 0; i < wave; ++i) {
                hole_at += red[kSelWaves + i];
                mover_at += red[2 * kSelWaves + i];
            }
        }
    }
    __syncthreads();  // the lists are whole
    int total = 0;
    for (int i = 0; i < kSelWaves; ++i) total += red[kSelWaves + i];
    for (int i = tid; i < total; i += kSelThreads) {
        const int to = hole_list[i], src = mover_list[i];
        ow[to] = w[src];
        op[to] = pos[src];
    }
    if (tid == 0) a.num_moves[blockIdx.x] = total;
}

// K and V rows of the listed moves; a.move_wgs neighbouring workgroups share one (sequence, kv head)'s list.
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictArgs a) {
    const int unit = blockIdx.x / a.move_wgs, part_wg = blockIdx.x % a.move_wgs, b = unit / a.Hkv, h = unit % a.Hkv;
    const int moves = a.num_moves[unit];
    const int32_t* hole_list = a.moves + (size_t)unit * 2 * a.max_moves;
    const int32_t* mover_list = hole_list + a.max_moves;
    const int64_t* table = a.table + (size_t)b * a.max_blocks;
    const int64_t work = (int64_t)moves * a.row_vecs;
    for (int64_t v = (int64_t)part_wg * kMoveThreads + threadIdx.x; v < work; v += (int64_t)a.move_wgs * kMoveThreads) {
        const int i = (int)(v / a.row_vecs), part = (int)(v % a.row_vecs);
        const int to = hole_list[i], src = mover_list[i];
        const size_t dst = (((size_t)table[to / a.bs] * a.Hkv + h) * a.bs + to % a.bs) * a.row_vecs + part;
        const size_t from = (((size_t)table[src / a.bs] * a.Hkv + h) * a.bs + src % a.bs) * a.row_vecs + part;
        const uint4 k = a.kc[from], x = a.vc[from];
        a.kc[dst] = k;
        a.vc[dst] = x;
    }
}

}  // namespace

hipError_t launch_kv_evict(const EvictArgs& a, hipStream_t stream) {
    if (a.B == 0) return hipSuccess;
    const size_t lds = (size_t)a.lds_keys * sizeof(uint32_t);
    evict_select_kernel<<<a.B * a.Hkv, kSelThreads, lds, stream>>>(a);
    if (hipError_t e = hipGetLastError()) return e;
    if (a.max_moves > 0) {
        evict_move_kernel<<<a.B * a.Hkv * a.move_wgs, kMoveThreads, 0, stream>>>(a);
        return hipGetLastError();
    }
    return hipSuccess;
}

}  // namespace kyro
