// The kernel that walks the lists of shared_attention.hip, instantiated in a translation unit for each group of head
// dims (shared_attention_bf16.hip, _wide.hip, _f32.hip) so that they compile in parallel.
//
// A workgroup of four waves takes its units one after the other: 128 query rows of one kv head, 32 a wave, over a range
// of tiles. Tiles are copied to LDS straight from the paged cache (buffer_load ... lds). The loop is a pipeline of three
// tiles: while the weights of tile i are worked out from its scores, the products of tile i + 1's scores run, and
// while its maxima are found, those of tile i's output; K of tile i + 2 and V of tile i + 1 are on their way. A wave alone
// on its SIMD then has something for the matrix unit at any time but at its barriers.
//
// Cycles of a tile of 64 tokens for a wave (64 sequences of 8 rows, all tokens common, head dim 128, two workgroups a CU): 32
// products of 32 each, 1024; 32 exponentials of 16 and 108 other vector operations of 4, 950. A step takes 2100 in the
// workgroup that is first, 2900 in the other; the copies never make it wait. Counters over 32768 common tokens (275 GFLOP,
// 285 us, 0.97 PFLOP/s at a clock that has fallen to 1.86 GHz): matrix units busy in 0.50 of the cycles, vector operations
// issued in 0.50, LDS active in 0.25 without a bank conflict. Other orders of the products (both halves' scores in turn
// before the outputs) and more operands in flight were level. 8 rows beside 100 to 1500 own tokens: 0.24, 0.30, 0.12 and
// 3.7 TB/s from memory; what waits there is the latency of own tokens' tiles, of which a workgroup has one on its way.
// In bf16 a weight is rounded once, to the 8 bits that the second product takes, as in the other attention kernels: an output
// is off by at most 2^-8 of its terms' size (rms 1.0e-3 of the outputs over 64 sequences behind 8192 tokens, beside 1.7e-3
// of an output's own rounding). The sum of the weights is of unrounded ones, in 32 bits like scores, outputs and states.
// What one unit takes beside its tiles (its entry, ids, K, first scores, state: 12 us alone) is hidden by the CU's other
// workgroup: loading all of the next unit's while the last tile is worked out changed nothing.
#pragma once

#include "common.hpp"
#include "kernels.hpp"
#include "prefill_tile.hpp"

namespace kyro {

namespace {

template <bool BF16, int DR>
__global__ __launch_bounds__(kPfThreads, shared_wgs_per_cu(BF16, DR)) void attn_shared_kernel(SharedArgs s) {
    using C = PfCfg<BF16, DR>;
    constexpr bool PIPE = shared_pipelined(BF16, DR);
    const AttnArgs& a = s.a;
    // An object for each buffer: the compiler's waits tell copies into one from reads of the other by the object.
    __shared__ uint4 sK0[C::NS * C::SLAB], sK1[C::NS * C::SLAB];
    __shared__ uint4 sV0[C::NS * C::SLAB], sV1[C::NS * C::SLAB];

    const int wg = (int)blockIdx.x / a.Hkv;
    const int kvh = (int)blockIdx.x - wg * a.Hkv;
    // Loads that follow from each other take 1 us each where the chip is cold, so the first unit comes with the range.
    const int used = s.head[0];
    const int4 range = s.starts[3 * wg], first0 = s.starts[3 * wg + 1], first1 = s.starts[3 * wg + 2];
    if (wg >= used) return;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31;
    const int h = lane >> 5;
    const bool younger = 2 * blockIdx.x >= gridDim.x;  // dispatched to a CU that has a workgroup
    const TileLane<C> at(lane);
    const float c = a.scale_log2;
    constexpr size_t kSlabBytes = (size_t)kPfBS * C::CPR * 16;
    const size_t head_off = (size_t)kvh * a.bs * (C::CPR * 16);

    for (int u = range.x; u <= range.y; ++u) {
        const bool first = u == range.x;
        const int4 e0 = first ? first0 : s.list[2 * (u + wg)], e1 = first ? first1 : s.list[2 * (u + wg) + 1];
        const int b = __builtin_amdgcn_readfirstlane(e0.x);
        if (b < 0) continue;  // this workgroup's share of the unit has no tile of it
        const int ctx = __builtin_amdgcn_readfirstlane(e0.w);
        const int row0 = __builtin_amdgcn_readfirstlane(e1.x);
        const int tile0 = __builtin_amdgcn_readfirstlane(e1.y);
        const bool common = __builtin_amdgcn_readfirstlane(e1.z) & kSharedAll;
        const int nt = __builtin_amdgcn_readfirstlane(e1.z) & ~kSharedAll;
        const int slot = __builtin_amdgcn_readfirstlane(e1.w);
        const bool causal = a.causal && !common;
        SeqInfo si;
        si.b = b;
        si.kvh = kvh;
        si.q0 = __builtin_amdgcn_readfirstlane(e0.y);
        si.q_len = __builtin_amdgcn_readfirstlane(e0.z);
        si.rows = si.q_len * a.group;
        si.ctx = ctx;
        const int wrow0 = row0 + 32 * wave;  // the wave's first row
        const int n = wrow0 + col;
        const int past = causal ? ctx - si.q_len + 1 : ctx;  // tokens row 0 sees
        // Rows past the unit take Q = 0 and every token; they are never stored.
        const int vis = n < si.rows && causal ? past + n / a.group : ctx;
        const int wave_lo = causal ? past + wrow0 / a.group : ctx;
        const int wg_hi = causal ? past + min(row0 + kPrefillRows - 1, si.rows - 1) / a.group : ctx;
        const int nslots = (max(wg_hi, 0) + kPfBS - 1) / kPfBS;  // slots the row group sees
        const bool active = wrow0 < si.rows;
        const int whole = max(wave_lo, 0) / C::TK - tile0;  // tiles that all the wave's rows see whole

        // Slab ids of 64 slots, one per lane (slab index of kv head 0, -1 for a bad block id), and of the next 64.
        constexpr int kFill = 64 / C::NS;
        auto load_ids = [&](int tile) -> int {
            const int x = tile * C::NS + lane;
            if (x >= nslots) return -1;
            const int blk = x / a.sub;
            const int64_t id = a.table[(size_t)b * a.max_blocks + blk];
            if (id < 0 || id >= a.num_blocks) {
                if (wave == 0) latch_error(a.err, ERR_BLOCK_ID);
                return -1;
            }
            return (int)id * a.Hkv * a.sub + (x - blk * a.sub);
        };
        int ids = load_ids(tile0);  // before the queries, which it would wait for
        int ids_next = 0;

        uint4 q[C::KS];
        {
            const char* qp = reinterpret_cast<const char*>(a.q) + out_row(a, si, n < si.rows ? n : 0) * (C::CPR * 16);
#pragma unroll
            for (int x = 0; x < C::KS; ++x) q[x] = n < si.rows ? load16(qp + (2 * x + h) * 16) : make_uint4(0, 0, 0, 0);
        }

        uint64_t bad = 0;
        auto slab_ptr = [&](const void* cache, int from, int i, int x) -> const void* {
            const int id = __builtin_amdgcn_readlane(from, (i % kFill) * C::NS + x);
            return id < 0 ? static_cast<const void*>(kPfZeroSlab) : static_cast<const char*>(cache) + id * kSlabBytes + head_off;
        };
        // With four slabs wave w copies slab w of K and of V, with two waves 0 and 1 those of K, 2 and 3 those of V.
        auto copy_lane = [&] {
            int x = lane;
            // Wide rows take many copies, whose offsets would stay in registers over the whole loop.
            if constexpr (!PIPE) asm volatile("" : "+v"(x));
            return x;
        };
        auto issue_k = [&](int i, int from, uint4* k) {
            if (C::NS == 4 || wave < 2) copy_slab<C, false, kLoadCached>(k + wave * C::SLAB, slab_ptr(a.k, from, i, wave), copy_lane());
        };
        auto issue_v = [&](int i, uint4* v) {
            const int x = C::NS == 4 ? wave : wave - 2;
            if (C::NS == 4 || wave >= 2) copy_slab<C, true, kLoadCached>(v + x * C::SLAB, slab_ptr(a.v, ids, i, x), copy_lane());
        };
        auto landed = [&] {
            __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's copies
            __syncthreads();                     // everyone's; and everyone is done with the tile before
        };

        f32x16 o[C::DT], S[C::TT], T[C::TT];
        float m = kNegInf, l = 0.f;  // running maximum, the lane's share of the row sum
#pragma unroll
        for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;

        // Scores of tile i that a row does not see, or that belong to a bad block, become -infinity.
        auto mask = [&](int i, uint32_t tbad, f32x16* x) {
            const int seen = vis - (tile0 + i) * C::TK - 4 * h;  // tokens from the lane's first one on
#pragma unroll
            for (int tt = 0; tt < C::TT; ++tt)
#pragma unroll
                for (int y = 0; y < 16; ++y) {
                    const bool ok = 32 * tt + 8 * (y / 4) + y % 4 < seen && !((tbad >> (2 * tt + y / 8)) & 1u);
                    x[tt][y] = ok ? x[tt][y] : kNegInf;
                }
        };
        auto row_max = [&](const f32x16* x) -> float {
            float r = x[0][0];
#pragma unroll
            for (int tt = 0; tt < C::TT; ++tt)
#pragma unroll
                for (int y = 0; y < 16; ++y) r = fmaxf(r, x[tt][y]);
            const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(r), __float_as_uint(r), false, false);
            return fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
        };
        auto tile_bad = [&](int i) -> uint32_t { return (uint32_t)(bad >> ((i % kFill) * C::NS)) & ((1u << C::NS) - 1u); };

        // The running maximum (scaled in bf16) with tile's maximum mx. No weight passes 1, so O^T cannot overflow before the
        // result does; over long contexts few tiles raise it for any of the wave's rows, and the others leave O^T and l alone.
        auto raise = [&](float mx) {
            const float top = fmaxf(m, BF16 ? mx * c : mx);
            if (!__any(top > m)) return;
            const float f = m == kNegInf ? 0.f : fast_exp2(BF16 ? m - top : (m - top) * c);
#pragma unroll
            for (int dt = 0; dt < C::DT; ++dt) o[dt] *= f;
            l *= f;
            m = top;
        };
        // Weight of a score, relative to ref.
        auto weight = [&](float x, float ref) { return fast_exp2(BF16 ? __builtin_fmaf(x, c, -ref) : (x - ref) * c); };
        // Tile i, whose scores are in S: its weights and its output.
        auto step = [&](int i, const uint4* vb, uint32_t tbad, f32x16* S) {
            if (i >= whole || tbad) mask(i, tbad, S);
            raise(row_max(S));
            const float ref = m == kNegInf ? 0.f : m;
#pragma unroll
            for (int tt = 0; tt < C::TT; ++tt) {
                float pt[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int y = 0; y < 16; ++y) {
                    S[tt][y] = weight(S[tt][y], ref);
                    pt[y % 4] += S[tt][y];
                }
                l += (pt[0] + pt[1]) + (pt[2] + pt[3]);
                uint4 w[2];
                if constexpr (BF16) tile_weights(S[tt], w);
                if constexpr (!BF16) __builtin_amdgcn_sched_barrier(0);  // V's reads stay below (registers)
                tile_output<C>(reinterpret_cast<const char*>(vb), S[tt], w, at, o, tt);
            }
        };
        // The same, with the scores of tile i + 1 (K at kb), which go to `next`; mx is the maximum of either
        // tile's scores before any mask. The order is written out: a product, the read of the operand kRing products
        // later, and some of the vector work, in turn (left to itself the compiler reads each operand right before
        // its product and keeps the work apart from both). `copy` issues one of the wave's 2 * kSlabCopies copies for
        // the tiles to come: all at once after the barrier, four waves' copies take the address unit 500 cycles, in
        // which no wave has a product to run.
        auto step_ahead = [&](int i, const uint4* kbuf, const uint4* vbuf, uint32_t tbad, float& mx, f32x16* S, f32x16* next,
                              auto&& copy) {
            if constexpr (PIPE) {
                static_assert(C::TT == 2, "two halves of a tile");
                const char* kb = reinterpret_cast<const char*>(kbuf);
                const char* vb = reinterpret_cast<const char*>(vbuf);
                if (i >= whole || tbad) {
                    mask(i, tbad, S);
                    mx = row_max(S);
                }
                raise(mx);
                const float ref = m == kNegInf ? 0.f : m;
                constexpr int NA = C::KS, NB = 2 * C::DT, kOps = 2 * (NA + NB), kRing = 4, kCopies = 2 * (C::SLAB / 64);
                // Products in order: scores of the next tile's first half, output of this one's first half, then the second.
                auto read = [&](int x) -> uint4 {
                    const int tt = x / (NA + NB), y = x % (NA + NB);
                    return y < NA ? k_operand<C>(kb, at, tt, y) : v_operand<C>(vb, at, tt, (y - NA) / C::DT, (y - NA) % C::DT);
                };
                uint4 ring[kRing], w[2][2];
                float pt[4] = {0.f, 0.f, 0.f, 0.f};
                float top = kNegInf;
                auto weigh = [&](int tt, int from, int to) {
#pragma unroll
                    for (int y = from; y < to; ++y) {
                        S[tt][y] = weight(S[tt][y], ref);
                        pt[y % 4] += S[tt][y];
                        if (y % 2) {
                            const uint32_t pair = pack_bf16x2(S[tt][y - 1], S[tt][y]);
                            uint4& to4 = w[tt][y / 8];
                            (y % 8 == 1 ? to4.x : y % 8 == 3 ? to4.y : y % 8 == 5 ? to4.z : to4.w) = pair;
                        }
                    }
                };
                auto most = [&](int tt, int from, int to) {
#pragma unroll
                    for (int y = from; y < to; ++y) top = fmaxf(top, next[tt][y]);
                };
#pragma unroll
                for (int x = 0; x < kRing; ++x) ring[x] = read(x);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int x = 0; x < kOps; ++x) {
                    const int tt = x / (NA + NB), y = x % (NA + NB);
                    if (y < NA) {
                        f32x16 zero;
#pragma unroll
                        for (int e = 0; e < 16; ++e) zero[e] = 0.f;
                        next[tt] = mfma_bf16(ring[x % kRing], q[y], y == 0 ? zero : next[tt]);
                    } else {
                        const int z = y - NA;
                        o[z % C::DT] = mfma_bf16(ring[x % kRing], w[tt][z / C::DT], o[z % C::DT]);
                    }
                    if (x + kRing < kOps) ring[x % kRing] = read(x + kRing);
                    if ((x + 1) * kCopies / kOps > x * kCopies / kOps) copy(x * kCopies / kOps);
                    // Weights of the first half beside the next one's scores, of the second beside the first's output and
                    // the next second's scores; maxima beside what is left.
                    if (tt == 0 && y < NA) weigh(0, 16 * y / NA, 16 * (y + 1) / NA);
                    if (tt == 0 && y >= NA) weigh(1, 8 * (y - NA) / NB, 8 * (y - NA + 1) / NB);
                    if (tt == 1 && y < NA) weigh(1, 8 + 8 * y / NA, 8 + 8 * (y + 1) / NA), most(0, 16 * y / NA, 16 * (y + 1) / NA);
                    if (tt == 1 && y >= NA + NB / 2) most(1, 16 * (y - NA - NB / 2) / (NB - NB / 2), 16 * (y - NA - NB / 2 + 1) / (NB - NB / 2));
                    __builtin_amdgcn_sched_barrier(0);
                }
                l += (pt[0] + pt[1]) + (pt[2] + pt[3]);
                const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
                mx = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
            }
        };

        // The slots of the last block past the context hold anything: V there becomes 0, so that it cannot reach O
        // through a zero weight.
        const int tail_tile = (ctx % kPfBS != 0 && nslots * kPfBS > ctx) ? ctx / C::TK : -1;
        auto clear_tail = [&](int i, uint4* v) {
            if (tile0 + i != tail_tile) return;
            const int t0 = ctx % kPfBS, slab = ctx % C::TK / kPfBS;
            for (int x = threadIdx.x; x < (kPfBS - t0) * C::NCH; x += kPfThreads) {
                const int t = t0 + x / C::NCH, pos = x % C::NCH;
                v[slab * C::SLAB + pos / C::CW * (kPfBS * C::CW) + t * C::CW + pos % C::CW] = make_uint4(0, 0, 0, 0);
            }
            __syncthreads();
        };
        auto next_ids = [&](int i) {  // before the copies of tile i > 0
            if (i % kFill != 0) return;
            ids = ids_next;
            bad = __ballot(ids < 0);
            ids_next = load_ids(tile0 + i + kFill);
        };

        __syncthreads();  // everyone has left the unit before
        if (nt > 0) {
            ids_next = nt > kFill ? load_ids(tile0 + kFill) : 0;
            bad = __ballot(ids < 0);
            issue_k(0, ids, sK0);
            issue_v(0, sV0);
            if constexpr (PIPE) {
                float mx = kNegInf;
                constexpr int kSlabCopies = C::SLAB / 64;
                // Tile i of nt: after the wait V of it is in v0 and K of the next in k1; V of the next goes to v1, K of
                // the one after that to k0.
                auto turn = [&](int i, uint4* k0, uint4* k1, uint4* v0, uint4* v1, f32x16* now, f32x16* next) {
                    // The two workgroups of a CU take turns at being first: left alone the older one is, and the other one
                    // still runs when it has ended (2048 rows a kv head over 32768 common tokens: 309 us for 319).
                    if (younger == (now == S)) __builtin_amdgcn_s_setprio(1);
                    else __builtin_amdgcn_s_setprio(0);
                    landed();
                    clear_tail(i, v0);
                    const uint32_t tbad = tile_bad(i);
                    next_ids(i + 1);
                    const auto vr = slab_buffer<C>(slab_ptr(a.v, ids, i + 1, wave));
                    const auto kr = slab_buffer<C>(slab_ptr(a.k, (i + 2) % kFill == 0 ? ids_next : ids, i + 2, wave), i + 2 >= nt);
                    auto copy = [&](int e) {
                        if (e < kSlabCopies) copy_chunks<C, true, kLoadCached>(v1 + wave * C::SLAB, vr, lane, e);
                        else copy_chunks<C, false, kLoadCached>(k0 + wave * C::SLAB, kr, lane, e - kSlabCopies);
                    };
                    if (active) {
                        step_ahead(i, k1, v0, tbad, mx, now, next, copy);
                    } else {
#pragma unroll
                        for (int e = 0; e < 2 * kSlabCopies; ++e) copy(e);
                    }
                };
                // The first scores wait for K of the first tile alone: the copies behind it are one slab, or two.
                static_assert(!PIPE || (C::NS == 4 && 2 * kSlabCopies < 16), "copies of a wave, in the wait's low bits");
                if (nt > 1) {
                    issue_k(1, ids, sK1);
                    __builtin_amdgcn_s_waitcnt(0x0f70 + 2 * kSlabCopies);
                } else {
                    __builtin_amdgcn_s_waitcnt(0x0f70 + kSlabCopies);
                }
                // A barrier alone: __syncthreads() would wait for all copies. What it orders is LDS that copies wrote and
                // that the wait above has seen land.
                asm volatile("" ::: "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                if (active) {
#pragma unroll
                    for (int tt = 0; tt < C::TT; ++tt) S[tt] = tile_scores<C>(reinterpret_cast<const char*>(sK0), q, at, tt);
                    mx = row_max(S);
                }
                int i = 0;
                while (true) {
                    if (i + 1 >= nt) break;
                    turn(i++, sK0, sK1, sV0, sV1, S, T);
                    if (i + 1 >= nt) {
#pragma unroll
                        for (int tt = 0; tt < C::TT; ++tt) S[tt] = T[tt];
                        break;
                    }
                    turn(i++, sK1, sK0, sV1, sV0, T, S);
                }
                landed();
                uint4* v = i % 2 ? sV1 : sV0;
                clear_tail(i, v);
                if (active) step(i, v, tile_bad(i), S);
            } else {
                // Registers hold one tile's scores: both operands of the next tile land while this one is computed.
                auto turn = [&](int i, uint4* k0, uint4* v0, uint4* k1, uint4* v1) {
                    landed();
                    clear_tail(i, v0);
                    const uint32_t tbad = tile_bad(i);
                    if (i + 1 < nt) {
                        next_ids(i + 1);
                        issue_k(i + 1, ids, k1);
                        issue_v(i + 1, v1);
                    }
                    if (!active) return;
#pragma unroll
                    for (int tt = 0; tt < C::TT; ++tt) S[tt] = tile_scores<C>(reinterpret_cast<const char*>(k0), q, at, tt);
                    step(i, v0, tbad, S);
                };
                for (int i = 0;;) {
                    turn(i, sK0, sV0, sK1, sV1);
                    if (++i >= nt) break;
                    turn(i, sK1, sV1, sK0, sV0);
                    if (++i >= nt) break;
                }
            }
        }

        auto store = [&] {
            float L = l + __shfl_xor(l, 32, 64);
            if (slot < 0) {
                const float inv = L > 0.f ? 1.f / L : 0.f;
                const size_t row = out_row(a, si, n);
#pragma unroll
                for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int d = 32 * dt + 8 * k + 4 * h;
                        if (C::D == DR || d < DR)
                            store_row4<DR>(a, row, d, o[dt][4 * k] * inv, o[dt][4 * k + 1] * inv, o[dt][4 * k + 2] * inv, o[dt][4 * k + 3] * inv);
                    }
                return;
            }
            // The part's state: m (scaled) and l by row, O^T in the order the lanes hold it (whole 1 KiB stores).
            const size_t wv = common ? ((size_t)slot * a.Hkv + kvh) * kPfWaves + wave
                                     : (size_t)s.tail_base + ((size_t)slot * a.Hkv + kvh) * s.tail_waves + wave;
            if constexpr (!BF16) {
                // Relative to the rounded scaled maximum that the merge weighs parts by.
                const float scaled = m * c;
                const float f = m == kNegInf ? 1.f : fast_exp2(__builtin_fmaf(m, c, -scaled));
                m = scaled;
                L *= f;
#pragma unroll
                for (int dt = 0; dt < C::DT; ++dt) o[dt] *= f;
            }
            if (h == 0) {
                a.ws_m[wv * 32 + col] = m;
                a.ws_l[wv * 32 + col] = L;
            }
#pragma unroll
            for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    reinterpret_cast<float4*>(a.ws_acc)[((wv * C::DT + dt) * 4 + k) * 64 + lane] =
                        make_float4(o[dt][4 * k], o[dt][4 * k + 1], o[dt][4 * k + 2], o[dt][4 * k + 3]);
        };
        if (n < si.rows) store();
    }
}

template <bool BF16, int DR>
void launch_shared_dim(const SharedArgs& s, hipStream_t stream) {
    attn_shared_kernel<BF16, DR><<<dim3((unsigned)(s.lanes * s.a.Hkv)), kPfThreads, 0, stream>>>(s);
}

}  // namespace

}  // namespace kyro
