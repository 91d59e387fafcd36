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
// evict_select_kernel: one workgroup a (sequence, kv head). Weights and positions are read once, 8 bytes a
// token (the positions a second time past 16 keys a thread), and the keys stay in registers, thread i holding
// slots i, i + 1024, .., for the three passes over 11, 11 and 10 bits (with 64 of them, past 32768 tokens, 151
// registers are spilled to scratch, and 1 with 32). The first digit holds the sign, the exponent and two bits of
// the mantissa, so weights that fall over many octaves spread over its bins. Ballots give each token its rank in
// slot order; the workgroup then copies its own K and V rows, up to kOwnMoves of them. evict_move_kernel: the
// rest, by many workgroups, where a call may have that many. Contexts past the registers read their keys again.
// What bounds it: latency (a dozen barriers, some five dependent loads) for few tokens, HBM for many moves, the
// one CU that selects for a (sequence, kv head) for long contexts (8 heads cut to a fifth: 27606 tokens 58 us,
// 52160 136 us, 131072, whose keys are read again for every pass, 444 us).
#include "common.hpp"
#include "kernels.hpp"

namespace kyro {
namespace {

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kBins = 2 * kSelThreads;
constexpr int kMoveThreads = 256;
constexpr int kMaxHeld = 64;   // keys a thread holds at most
constexpr int kOwnMoves = kEvictOwnMoves;

// Order-preserving bits: a < b as floats <=> rank(a) < rank(b); -0 ranks as +0, NaN as -infinity.
__device__ __forceinline__ uint32_t rank_bits(float w) {
    uint32_t u = __float_as_uint(w);
    u = (u & 0x7fffffffu) > 0x7f800000u ? 0xff800000u : u;
    u = u == 0x80000000u ? 0u : u;
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

struct Shared {
    int hist[kBins];
    int red[kSelWaves];
    int red2[kSelWaves];
    int found[2];
    int bad;
    // Tokens of one kind in each group of 64 slots, then how many there are before it.
    int count[2][kMaxHeld * kSelWaves];
    int hole[kOwnMoves], mover[kOwnMoves];  // the first of each list
    int4 move[kOwnMoves];                   // (block, slot) to, (block, slot) from
};

// Maximum over the workgroup; every thread gets it.
__device__ __forceinline__ int block_max(int v, int* red) {
    for (int m = 32; m; m >>= 1) v = max(v, __shfl_xor(v, m, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < kSelWaves; ++i) v = max(v, red[i]);
    return v;
}

// Exclusive sum over the workgroup's threads; *total gets the whole. red: of its own for each call in a row.
__device__ __forceinline__ int block_scan(int v, int* red, int* total) {
    const int incl = wave_incl_scan_i(v), wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 63) red[wave] = incl;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kSelWaves; ++i) {
        const int x = red[i];
        before += i < wave ? x : 0;
        all += x;
    }
    *total = all;
    return before + incl - v;
}

// Notes what is wrong with the sequence's block ids (n of its tokens are known to fit); read behind a barrier.
__device__ __forceinline__ void check_blocks(const EvictArgs& a, int b, int n, Shared& sh) {
    int bad = 0;
    for (int i = threadIdx.x; i < (n + a.bs - 1) / a.bs; i += kSelThreads) {
        const int64_t id = a.table[(size_t)b * a.max_blocks + i];
        if (id < 0 || id >= a.num_blocks) bad = ERR_BLOCK_ID;
    }
    if (bad) atomicOr(&sh.bad, bad);
}

// One (sequence, kv head)'s arrays.
struct Unit {
    const float* w;
    const int32_t* pos;
    float* ow;
    int32_t* op;
    int n, budget, sink, from;  // positions above `from` are protected
    int32_t* holes;  // the lists' entries from own_moves on
    int32_t* movers;
    __device__ __forceinline__ void protect(int newest, int recent) { from = (int)max((int64_t)newest - recent, (int64_t)INT32_MIN); }
    __device__ __forceinline__ uint32_t key(int p, float x) const { return ((p < sink) | (p > from)) ? 0xffffffffu : rank_bits(x); }
};

// Entry i of a list: the first ones in LDS, those that the other kernel reads in memory.
__device__ __forceinline__ void list(const EvictArgs& a, int* first, int32_t* rest, int i, int t) {
    if (i < kOwnMoves) first[i] = t;
    if (i >= a.own_moves) rest[i] = t;
}

// Marks the kept tokens and lists holes and movers; R keys a thread (R = 0: any number, read again). Returns
// the number of moves, or -1 (before anything is written) for a sequence with a bad block.
template <int R>
__device__ __forceinline__ int select(const EvictArgs& a, int b, Unit u, Shared& sh) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    constexpr int kHeld = R ? R : 1;
    uint32_t key[kHeld];
    const int rounds = R ? R : (u.n + kSelThreads - 1) / kSelThreads;
    int newest = INT32_MIN;
    if constexpr (R > 0 && R <= 16) {
        int p[kHeld];
        float x[kHeld];
#pragma unroll
        for (int r = 0; r < kHeld; ++r) {
            // Behind the last token it again: a load that is always made waits for nothing.
            const int t = min(r * kSelThreads + tid, u.n - 1);
            p[r] = u.pos[t];
            x[r] = u.w[t];
        }
        check_blocks(a, b, u.n, sh);  // while they are under way
#pragma unroll
        for (int r = 0; r < kHeld; ++r) newest = max(newest, p[r]);
        newest = block_max(newest, sh.red);
        u.protect(newest, a.recent);
#pragma unroll
        for (int r = 0; r < kHeld; ++r) key[r] = u.key(p[r], x[r]);
    } else {
        check_blocks(a, b, u.n, sh);
#pragma unroll 16
        for (int r = 0; r < rounds; ++r) {
            newest = max(newest, u.pos[min(r * kSelThreads + tid, u.n - 1)]);
        }
        newest = block_max(newest, sh.red);
        u.protect(newest, a.recent);
        if constexpr (R > 0) {  // positions again, from L2: held beside the keys they would not fit
#pragma unroll
            for (int r = 0; r < kHeld; ++r) {
                const int t = min(r * kSelThreads + tid, u.n - 1);
                key[r] = u.key(u.pos[t], u.w[t]);
                // A part at a time, so that not all the loads come first: the keys fill the registers as it is.
                if (r % (R == 32 ? 16 : 8) == (R == 32 ? 15 : 7)) __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    if (sh.bad) return -1;  // block_max had a barrier
    const auto key_at = [&](int r) -> uint32_t {
        if constexpr (R > 0) return key[r];
        const int t = r * kSelThreads + tid;
        return t < u.n ? u.key(u.pos[t], u.w[t]) : 0u;
    };

    // The budget-th largest key, digit by digit from the top; `want` counts within the keys that share the
    // digits found so far. Thread i owns the bins 2 i and 2 i + 1 from the largest down, and leaves them empty.
    uint32_t T = 0;
    int want = u.budget;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, above = pass == 0 ? 32 : pass == 1 ? 21 : 10;
        const uint32_t mask = pass == 2 ? 1023u : 2047u;
        const auto count = [&](uint32_t k, int t) {
            if (t < u.n && (pass == 0 || (k >> above) == T)) atomicAdd(&sh.hist[(k >> shift) & mask], 1);
        };
        if constexpr (R > 0) {
#pragma unroll
            for (int r = 0; r < kHeld; ++r) count(key[r], r * kSelThreads + tid);
        } else {
            for (int r = 0; r < rounds; ++r) count(key_at(r), r * kSelThreads + tid);
        }
        __syncthreads();
        const int hi = kBins - 1 - 2 * tid;
        const int c0 = sh.hist[hi], c1 = sh.hist[hi - 1];
        sh.hist[hi] = sh.hist[hi - 1] = 0;
        int total;
        const int before = block_scan(c0 + c1, pass == 1 ? sh.red2 : sh.red, &total);
        if (before < want && want <= before + c0 + c1) {
            const bool first = want <= before + c0;
            sh.found[0] = first ? hi : hi - 1;
            sh.found[1] = first ? before : before + c0;
        }
        __syncthreads();
        T = (T << (pass == 2 ? 10 : 11)) | (uint32_t)sh.found[0];
        want -= sh.found[1];
    }
    // `want` of the keys equal to T stay, those of the lowest slots.

    const unsigned long long below = lane == 0 ? 0ull : (~0ull >> (64 - lane));
    // Turns the counts of `rounds` x kSelWaves groups, in slot order, into how many come before each.
    const auto scan_counts = [&](int* count, int* red) -> int {
        int carry = 0;
        if constexpr (R > 0) {  // at most kSelThreads groups
            const int groups = kHeld * kSelWaves;
            const int v = tid < groups ? count[tid] : 0;
            int total;
            const int before = block_scan(v, red, &total);
            if (tid < groups) count[tid] = before;
            carry = total;
        }
        __syncthreads();
        return carry;
    };
    if constexpr (R > 0) {
#pragma unroll
        for (int r = 0; r < kHeld; ++r) {
            const bool in = r * kSelThreads + tid < u.n;
            const int c = __popcll(__ballot(in && key[r] == T));
            if (lane == 0) sh.count[0][r * kSelWaves + wave] = c;
        }
        __syncthreads();
        scan_counts(sh.count[0], sh.red2);
        unsigned long long kept = 0;  // bit r: this thread's r-th token stays
#pragma unroll
        for (int r = 0; r < kHeld; ++r) {
            const int t = r * kSelThreads + tid;
            const bool in = t < u.n;
            const unsigned long long ties = __ballot(in && key[r] == T);
            const int rank = sh.count[0][r * kSelWaves + wave] + __popcll(ties & below);
            const bool keep = in && (key[r] > T || (key[r] == T && rank < want));
            kept |= (unsigned long long)keep << r;
        }
        __syncthreads();  // the ties' ranks have been read
#pragma unroll
        for (int r = 0; r < kHeld; ++r) {
            const int t = r * kSelThreads + tid;
            const bool keep = (kept >> r) & 1;
            const int holes = __popcll(__ballot(!keep && t < u.budget)), movers = __popcll(__ballot(keep && t >= u.budget));
            if (lane == 0) {
                sh.count[0][r * kSelWaves + wave] = holes;
                sh.count[1][r * kSelWaves + wave] = movers;
            }
        }
        __syncthreads();
        const int moves = scan_counts(sh.count[0], sh.red);
        scan_counts(sh.count[1], sh.red2);
#pragma unroll
        for (int r = 0; r < kHeld; ++r) {
            const int t = r * kSelThreads + tid;
            const bool keep = (kept >> r) & 1, hole = !keep && t < u.budget, mover = keep && t >= u.budget;
            const unsigned long long hb = __ballot(hole), mb = __ballot(mover);
            if (hole) list(a, sh.hole, u.holes, sh.count[0][r * kSelWaves + wave] + __popcll(hb & below), t);
            if (mover) list(a, sh.mover, u.movers, sh.count[1][r * kSelWaves + wave] + __popcll(mb & below), t);
        }
        if ((u.ow != u.w) | (u.op != u.pos)) {  // out of place: what stays where it is, four loads at a time
#pragma unroll 1
            for (int r0 = 0; r0 < kHeld && r0 * kSelThreads < u.budget; r0 += 4) {
                float x[4];
                int p[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int t = min((r0 + j) * kSelThreads + tid, u.n - 1);
                    x[j] = u.w[t];
                    p[j] = u.pos[t];
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int t = (r0 + j) * kSelThreads + tid;
                    if (t < u.budget && ((kept >> (r0 + j)) & 1)) {
                        if (u.ow != u.w) u.ow[t] = x[j];
                        if (u.op != u.pos) u.op[t] = p[j];
                    }
                }
            }
        }
        return moves;
    } else {
        // Round by round, each with its own ranks: ties before, holes before, movers before.
        int ties_before = 0, holes_before = 0, movers_before = 0;
        for (int r = 0; r < rounds; ++r) {
            const int t = r * kSelThreads + tid;
            const bool in = t < u.n;
            const uint32_t k = key_at(r);
            int total;
            __syncthreads();  // the round before has read its sums
            const int rank = ties_before + block_scan(in && k == T, sh.red, &total);
            ties_before += total;
            const bool keep = in && (k > T || (k == T && rank < want));
            const bool hole = in && !keep && t < u.budget, mover = keep && t >= u.budget;
            const int at = block_scan(hole | (mover << 16), sh.red2, &total);
            if (hole) list(a, sh.hole, u.holes, holes_before + (at & 0xffff), t);
            if (mover) list(a, sh.mover, u.movers, movers_before + (at >> 16), t);
            holes_before += total & 0xffff;
            movers_before += total >> 16;
            if (keep && !mover) {
                if (u.ow != u.w) u.ow[t] = u.w[t];
                if (u.op != u.pos) u.op[t] = u.pos[t];
            }
        }
        return holes_before;
    }
}

// HELD: most keys a thread holds (4, 16, 32, 64), which sets the kernel's registers; with 4, two workgroups share
// a CU (64 x 2304 tokens of 8 heads: 50 us with one, 43 with two).
template <int HELD>
__global__ __launch_bounds__(kSelThreads, HELD == 4 ? 8 : 4) void evict_select_kernel(EvictArgs a) {
    __shared__ Shared sh;
    const int b = blockIdx.x / a.Hkv, h = blockIdx.x % a.Hkv;
    const int tid = threadIdx.x;
    const int64_t n64 = a.ctx_lens[b];
    const int64_t row = a.state_rows ? a.state_rows[b] : b;
    if (tid == 0) sh.bad = 0;
    for (int i = tid; i < kBins; i += kSelThreads) sh.hist[i] = 0;
    if (tid == 0) {
        a.num_moves[blockIdx.x] = 0;
        if (h == 0) a.out_ctx_lens[b] = n64 > a.budget && n64 <= a.cap ? a.budget : n64;
    }
    int bad = n64 < 0 || n64 > a.cap ? ERR_CTX_LEN : 0;
    if (a.state_rows) {
        bad |= row < 0 || row >= a.num_state_rows ? ERR_STATE_ROW : 0;
        int twice = 0;
        for (int i = tid; i < a.B; i += kSelThreads)
            if (i != b && a.state_rows[i] == row) twice = 1;
        if (__syncthreads_or(twice)) bad |= ERR_STATE_ROW;
    }
    if (bad) {
        if (tid == 0) {
            latch_error(a.err, bad);
            if (h == 0) a.out_ctx_lens[b] = n64;
        }
        return;
    }
    const size_t base = ((size_t)row * a.Hkv + h) * a.max_tokens;
    Unit u = {a.weights + base, a.positions + base, a.out_weights + base, a.out_positions + base, (int)n64, a.budget, a.sink, 0,
              a.moves + (size_t)blockIdx.x * 2 * a.max_moves, a.moves + ((size_t)blockIdx.x * 2 + 1) * a.max_moves};
    if (u.n <= u.budget) {
        for (int t = tid; t < u.n; t += kSelThreads) {
            if (u.ow != u.w) u.ow[t] = u.w[t];
            if (u.op != u.pos) u.op[t] = u.pos[t];
        }
        return;
    }
    __syncthreads();
    const int rounds = (u.n + kSelThreads - 1) / kSelThreads;
    int moves;
    if (rounds <= 1) moves = select<1>(a, b, u, sh);
    else if (rounds <= 4) moves = select<4>(a, b, u, sh);
    else if (HELD >= 16 && rounds <= 16) moves = select<HELD >= 16 ? 16 : 1>(a, b, u, sh);
    else if (HELD >= 32 && rounds <= 32) moves = select<HELD >= 32 ? 32 : 1>(a, b, u, sh);
    else if (HELD >= 64 && rounds <= 64) moves = select<HELD >= 64 ? 64 : 1>(a, b, u, sh);
    else moves = select<0>(a, b, u, sh);
    if (moves < 0) {
        if (tid == 0) {
            latch_error(a.err, sh.bad);
            if (h == 0) a.out_ctx_lens[b] = n64;
        }
        return;
    }
    __syncthreads();  // the lists are whole
    const int64_t* table = a.table + (size_t)b * a.max_blocks;
    const int own = min(moves, a.own_moves);
    for (int i = tid; i < moves; i += kSelThreads) {
        const int to = i < kOwnMoves ? sh.hole[i] : u.holes[i], src = i < kOwnMoves ? sh.mover[i] : u.movers[i];
        if (i < own) {
            const int p = to / a.bs, q = src / a.bs;
            sh.move[i] = make_int4((int)table[p], to - p * a.bs, (int)table[q], src - q * a.bs);
        }
        const float x = u.w[src];
        const int p = u.pos[src];
        u.ow[to] = x;
        u.op[to] = p;
    }
    __syncthreads();
    const int vecs = own * a.row_vecs;
    const size_t head = (size_t)h * a.bs;
    for (int v = tid; v < vecs; v += kSelThreads) {
        const int i = v / a.row_vecs, part = v - i * a.row_vecs;
        const int4 m = sh.move[i];
        const size_t dst = ((size_t)m.x * a.Hkv * a.bs + head + m.y) * a.row_vecs + part;
        const size_t from = ((size_t)m.z * a.Hkv * a.bs + head + m.w) * a.row_vecs + part;
        const uint4 k = a.kc[from], x = a.vc[from];
        a.kc[dst] = k;
        a.vc[dst] = x;
    }
    if (tid == 0) a.num_moves[blockIdx.x] = moves;
}

// K and V rows of the moves that the selection has left; a.move_wgs neighbouring workgroups share one
// (sequence, kv head)'s list.
__device__ __forceinline__ size_t row_of(const EvictArgs& a, const int64_t* table, int h, int t) {
    const int page = t / a.bs;
    return (((size_t)table[page] * a.Hkv + h) * a.bs + (t - page * a.bs)) * a.row_vecs;
}
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictArgs a) {
    const int unit = blockIdx.x / a.move_wgs, part_wg = blockIdx.x % a.move_wgs, b = unit / a.Hkv, h = unit % a.Hkv;
    const int moves = a.num_moves[unit];
    const int32_t* hole_list = a.moves + (size_t)unit * 2 * a.max_moves;
    const int32_t* mover_list = hole_list + a.max_moves;
    const int64_t* table = a.table + (size_t)b * a.max_blocks;
    const int64_t work = (int64_t)moves * a.row_vecs;
    for (int64_t v = (int64_t)a.own_moves * a.row_vecs + (int64_t)part_wg * kMoveThreads + threadIdx.x; v < work;
         v += (int64_t)a.move_wgs * kMoveThreads) {
        const int i = (int)(v / a.row_vecs), part = (int)(v - (int64_t)i * a.row_vecs);
        const size_t to = row_of(a, table, h, hole_list[i]) + part, src = row_of(a, table, h, mover_list[i]) + part;
        const uint4 k = a.kc[src], x = a.vc[src];
        a.kc[to] = k;
        a.vc[to] = x;
    }
}

}  // namespace

hipError_t launch_kv_evict(const EvictArgs& a, hipStream_t stream) {
    if (a.B == 0) return hipSuccess;
    const int units = a.B * a.Hkv;
    if (a.cap <= 4 * kSelThreads) evict_select_kernel<4><<<units, kSelThreads, 0, stream>>>(a);
    else if (a.cap <= 16 * kSelThreads) evict_select_kernel<16><<<units, kSelThreads, 0, stream>>>(a);
    else if (a.cap <= 32 * kSelThreads) evict_select_kernel<32><<<units, kSelThreads, 0, stream>>>(a);
    else evict_select_kernel<64><<<units, kSelThreads, 0, stream>>>(a);
    if (a.max_moves > a.own_moves) evict_move_kernel<<<units * a.move_wgs, kMoveThreads, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace kyro
