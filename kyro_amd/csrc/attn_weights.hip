// Accumulated attention weight of cached tokens (gfx950): for each kv head and cached token t,
//     w[t] += sum over the step's query rows r of that head's group of  exp(s[r,t] - m[r]) / l[r],
//     s[r,t] = scale q_r . k_t over the tokens r sees,  m[r] = max_t s,  l[r] = sum_t exp(s - m).
//
// The sum over rows needs every row's m and l first, so there are two passes:
//   stats   m and l of each row over a chunk of tokens, one running maximum and sum per lane;
//   sum     adds up exp2(s - (m + log l)) per token, with m and l merged over the chunks.
// Between them a score is either kept (4 bytes a row and token, written once and read once) or computed
// again from the keys (D elements a token, whatever the rows): decode steps of a few rows keep, verify steps
// and prompts compute. One wave owns a token's sum and adds rows in order: no atomics, the same result
// every time.
//
// The products run on MFMA. Both operands of a 16x16x32 product hold 8 elements of row lane % 16 from
// element 8 (lane / 16), so keys and queries go from memory straight into them, 16 bytes a lane, whatever
// the block size; the result has the first operand's index in the lane's four registers and the second's
// in the lane. The f32 caches take 16x16x4 products on 4-element pieces, the same pieces for both operands.
#include <cfloat>
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"

namespace kyro {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

// Part i of 16 rows as an operand: 32 of their elements, 8 a lane. A product does not mind which elements
// its k steps take as long as both operands take the same, so a lane's 16-byte pieces are chosen for the
// loads: lanes l, l + 16, l + 32 and l + 48 share row l % 16, and two pieces of 32 adjacent bytes each (the
// next part's, or the f32 part's other half) make every load touch all of its rows' 128-byte lines.
// `last`: there is no next part to share a line with. FULL: the row has all of its elements, else D bounds
// them and the rest are 0.
template <bool BF16>
struct Frag;
template <>
struct Frag<true> {
    bf16x8 x;
    template <bool FULL>
    __device__ __forceinline__ void load(const void* base, size_t row, int i, bool last, int D, int lane) {
        const int at = piece(i, last, 0, lane);
        const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + row;
        uint4 u = *reinterpret_cast<const uint4*>(p + (FULL || at < D ? at : 0));
        if (!FULL && at >= D) u = make_uint4(0, 0, 0, 0);
        x = __builtin_bit_cast(bf16x8, u);
    }
    __device__ __forceinline__ void get(const uint4 (&p)[1][64], int lane) { x = __builtin_bit_cast(bf16x8, p[0][lane]); }
    __device__ __forceinline__ void put(uint4 (&p)[1][64], int lane) const { p[0][lane] = __builtin_bit_cast(uint4, x); }
    // Element of the row that piece p of part i starts with.
    static __device__ __forceinline__ int piece(int i, bool last, int, int lane) {
        return last && i % 2 == 0 ? 32 * i + 8 * (lane >> 4) : 64 * (i / 2) + 16 * (lane >> 4) + 8 * (i % 2);
    }
    __device__ __forceinline__ void zero() { x = __builtin_bit_cast(bf16x8, make_uint4(0, 0, 0, 0)); }
    static __device__ __forceinline__ f32x4 mma(const Frag& a, const Frag& b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.x, b.x, c, 0, 0, 0);
    }
};
template <>
struct Frag<false> {
    f32x4 x[2];
    template <bool FULL>
    __device__ __forceinline__ void load(const void* base, size_t row, int part, bool, int D, int lane) {
        const float* p = reinterpret_cast<const float*>(base) + row;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int at = piece(part, false, i, lane);
            x[i] = *reinterpret_cast<const f32x4*>(p + (FULL || at < D ? at : 0));
            if (!FULL && at >= D) x[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    __device__ __forceinline__ void get(const uint4 (&p)[2][64], int lane) {
        x[0] = __builtin_bit_cast(f32x4, p[0][lane]);
        x[1] = __builtin_bit_cast(f32x4, p[1][lane]);
    }
    __device__ __forceinline__ void put(uint4 (&p)[2][64], int lane) const {
        p[0][lane] = __builtin_bit_cast(uint4, x[0]);
        p[1][lane] = __builtin_bit_cast(uint4, x[1]);
    }
    static __device__ __forceinline__ int piece(int i, bool, int p, int lane) { return 32 * i + 8 * (lane >> 4) + 4 * p; }
    __device__ __forceinline__ void zero() { x[0] = x[1] = f32x4{0.f, 0.f, 0.f, 0.f}; }
    static __device__ __forceinline__ f32x4 mma(const Frag& a, const Frag& b, f32x4 c) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.x[i][j], b.x[i][j], c, 0, 0, 0);
        return c;
    }
};

// A work item's sequence: found by walking the sequences in strips of 64, one a lane, with the items of
// each counted from its own length. Items of a workgroup rise, so the walk goes on where it was. Backwards,
// from the last sequence on, it goes over the keys of a pass in the other order: what was read last is
// still in the memory-side cache then.
struct Sequence {
    int b, q0, n;   // rows [q0, q0 + n)
    int ctx;
    int64_t first;  // the sequence's first item
};

struct Walk {
    int strip = -64;      // first sequence of the strip in the registers
    int64_t base = 0;     // items before the strip
    int total = 0;        // items of the strip
    int incl = 0, q0 = 0, n = 0, ctx = 0;

    // per_sequence(ctx, n): a sequence's items. Wave-uniform; false behind the last item.
    template <typename F>
    __device__ __forceinline__ bool find(const AttnWeightsArgs& a, bool backwards, int64_t item, F per_sequence, Sequence& s) {
        const int lane = threadIdx.x & 63;
        while (item >= base + total) {
            base += total;
            strip += 64;
            if (strip >= a.B) return false;
            const int b = backwards ? a.B - 1 - strip - lane : strip + lane;
            int count = 0;
            n = ctx = 0;
            if (b >= 0 && b < a.B) {
                int r0 = b, r1 = b + 1;
                if (a.q_start) {
                    r0 = a.q_start[b];
                    r1 = a.q_start[b + 1];
                }
                const int64_t c = a.ctx_lens[b];
                int bad = 0;
                if (r0 < 0 || r1 < r0 || r1 > a.total_q || r1 - r0 > a.max_q_len) bad |= ERR_Q_LAYOUT;
                else if (c < 0 || c > a.cap) bad |= ERR_CTX_LEN;
                if (bad) {
                    latch_error(a.err, bad);
                } else if (r1 > r0 && c > 0) {
                    q0 = r0;
                    n = r1 - r0;
                    ctx = (int)c;
                    count = per_sequence(ctx, n);
                }
            }
            incl = wave_incl_scan_i(count);
            total = __builtin_amdgcn_readlane(incl, 63);
        }
        const int at = (int)(item - base);
        const int l = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(incl > at)) - 1);
        s.b = backwards ? a.B - 1 - strip - l : strip + l;
        s.q0 = __builtin_amdgcn_readlane(q0, l);
        s.n = __builtin_amdgcn_readlane(n, l);
        s.ctx = __builtin_amdgcn_readlane(ctx, l);
        s.first = base + (l ? __builtin_amdgcn_readlane(incl, l - 1) : 0);
        return true;
    }
};

// A cached token's key is found in two steps, so that a block id is under way before it is looked at: a
// check right behind its load would hold up the keys that are loaded between.
__device__ __forceinline__ int page_of(const AttnWeightsArgs& a, int t) {
    return a.bs_shift >= 0 ? t >> a.bs_shift : t / a.bs;
}
__device__ __forceinline__ int64_t block_of(const AttnWeightsArgs& a, int b, int t) {
    return a.table[(size_t)b * a.max_blocks + page_of(a, t)];
}
// Element offset of token t in block blk of kv head h, or -1 for a bad block.
__device__ __forceinline__ int64_t key_offset(const AttnWeightsArgs& a, int64_t blk, int h, int t) {
    if (blk < 0 || blk >= a.num_blocks) {
        latch_error(a.err, ERR_BLOCK_ID);
        return -1;
    }
    const uint32_t in_block = (uint32_t)(h * a.bs + (t - page_of(a, t) * a.bs)) * (uint32_t)a.D;
    return (int64_t)((uint64_t)(uint32_t)blk * a.block_elems + in_block);
}

// r / group: group_magic is 2^32 / group rounded up, exact while r * group < 2^32.
__device__ __forceinline__ int step_row(const AttnWeightsArgs& a, int r) {
    return a.group == 1 ? r : (int)__umulhi((uint32_t)r, a.group_magic);
}

// Row r (of a kv head's n * group rows, row by row) in the query, counted in rows of D.
__device__ __forceinline__ size_t query_row(const AttnWeightsArgs& a, const Sequence& s, int h, int r) {
    const int j = step_row(a, r);
    return (size_t)(s.q0 + j) * a.H + (size_t)h * a.group + (r - j * a.group);
}

// The last token that row r sees.
__device__ __forceinline__ int last_seen(const AttnWeightsArgs& a, const Sequence& s, int r) {
    return a.causal ? s.ctx - s.n + step_row(a, r) : s.ctx - 1;
}

// A row at element off, or zeros for off < 0.
template <bool BF16, int STEPS, bool FULL>
__device__ __forceinline__ void load_row(Frag<BF16>* x, const void* base, int64_t off, int D, int lane) {
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        if (off >= 0) x[i].template load<FULL>(base, (size_t)off, i, i == STEPS - 1, D, lane);
        else x[i].zero();
    }
}

// The running (max, sum) of two sets of scores, in base 2. The sum that goes with a maximum of -infinity is
// 0, or NaN where a score was: that has to reach the result.
__device__ __forceinline__ void merge(float& m, float& l, float m2, float l2) {
    const float top = fmaxf(m, m2);
    l = l * (m == kNegInf ? 1.f : fast_exp2(m - top)) + l2 * (m2 == kNegInf ? 1.f : fast_exp2(m2 - top));
    m = top;
}

// m + log2 l, what a row's scores are set off against; infinity for a row that sees nothing, which then
// adds exp2(s - inf) = 0.
__device__ __forceinline__ float log_sum(float m, float l) {
    return m == kNegInf && l == 0.f ? -kNegInf : m + __builtin_amdgcn_logf(l);
}

// Adds N scores to a running (max, sum).
template <int N>
__device__ __forceinline__ void add_scores(float& m, float& l, const float (&x)[N]) {
    float top = m;
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, x[i]);
    const float ref = top == kNegInf ? 0.f : top;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) sum += fast_exp2(x[i] - ref);
    l = l * fast_exp2(m - ref) + sum;
    m = top;
}

// The same for N products that are scores once scaled (scale >= 0).
template <int N>
__device__ __forceinline__ void add_products(float& m, float& l, const float (&x)[N], float scale) {
    float most = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) most = fmaxf(most, x[i]);
    const float top = fmaxf(m, most * scale), ref = top == kNegInf ? 0.f : top;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) sum += fast_exp2(x[i] * scale - ref);
    l = l * fast_exp2(m - ref) + sum;
    m = top;
}

// The state row of a sequence's weights, or -1 (and an error) where the caller's is bad. Workgroup-uniform.
__device__ __forceinline__ int64_t state_row(const AttnWeightsArgs& a, int b) {
    if (!a.state_rows) return b;
    const int row = a.state_rows[b];
    int bad = row < 0 || row >= a.num_state_rows;
    for (int i = threadIdx.x; i < a.B; i += kThreads)
        if (i != b && a.state_rows[i] == row) bad = 1;
    if (!__syncthreads_or(bad)) return row;
    if (threadIdx.x == 0) latch_error(a.err, ERR_STATE_ROW);
    return -1;
}

// What token t < end has from the steps before: nothing for the step's own.
__device__ __forceinline__ float old_weight(const AttnWeightsArgs& a, const Sequence& s, size_t base, int t, int end) {
    return t < end && t < s.ctx - s.n ? a.w[base + t] : 0.f;
}

__device__ __forceinline__ void store_weight(const AttnWeightsArgs& a, const Sequence& s, size_t base, int t, float x) {
    const int old = s.ctx - s.n;
    a.out_w[base + t] = x;
    if (t >= old) a.positions[base + t] = a.row_pos ? (int32_t)a.row_pos[s.q0 + t - old] : t;
}

// Where the weights go elsewhere, a sequence that has no rows in the step takes its own along. The workgroups of
// the kernel that calls it share a sequence's tokens where they are more than the sequences; at its end, so that
// the work items' loads wait for nothing of this.
__device__ __forceinline__ void copy_idle(const AttnWeightsArgs& a) {
    const int parts = max(1u, gridDim.x / (unsigned)a.B);
    for (unsigned item = blockIdx.x; item < (unsigned)parts * a.B; item += gridDim.x) {
        const int part = (int)(item / (unsigned)a.B), b = (int)item - part * a.B;
        const int r0 = a.q_start[b];
        if (r0 != a.q_start[b + 1]) continue;
        const int64_t ctx = a.ctx_lens[b];
        const int bad = r0 < 0 || r0 > a.total_q ? ERR_Q_LAYOUT : ctx < 0 || ctx > a.cap ? ERR_CTX_LEN : 0;
        if (bad && threadIdx.x == 0) latch_error(a.err, bad);
        if (bad || ctx == 0) continue;
        const int64_t row = state_row(a, b);
        if (row < 0) continue;
        const int64_t per = (ctx + parts - 1) / parts, from = part * per, to = min(ctx, from + per);
        for (int h = 0; h < a.Hkv; ++h) {
            const size_t base = ((size_t)row * a.Hkv + h) * a.max_tokens;
            for (int64_t t = from + threadIdx.x; t < to; t += kThreads) a.out_w[base + t] = a.w[base + t];
        }
    }
}

// m + log2 l of a kv head's first N rows (a power of two, at most kThreads), merged over the chunks.
template <int N>
__device__ __forceinline__ void merge_chunks(const AttnWeightsArgs& a, const Sequence& s, int h, int parts, float2* partial,
                                             float* lse) {
    const int r = threadIdx.x % N, rows = s.n * a.group;
    float m = kNegInf, l = 0.f;
    if (r < rows) {
        const float2* p = a.part + query_row(a, s, h, r);
        for (int c = threadIdx.x / N; c < parts; c += kThreads / N) {
            const float2 x = p[(size_t)c * a.total_q * a.H];
            merge(m, l, x.x, x.y);
        }
    }
    __syncthreads();  // the item before has read lse
    partial[threadIdx.x] = make_float2(m, l);
    __syncthreads();
    if (threadIdx.x < N) {
        float2 x = partial[threadIdx.x];
        for (int i = 1; i < kThreads / N; ++i) merge(x.x, x.y, partial[i * N + threadIdx.x].x, partial[i * N + threadIdx.x].y);
        lse[threadIdx.x] = log_sum(x.x, x.y);
    }
    __syncthreads();
}

// ------------------------------------------------------------------- few rows (decode, verify)

// Item: (sequence, chunk of tokens, kv head). All rows of the head are in registers (16 NT of them), each wave
// takes a quarter of the chunk, U tiles of 16 tokens at a time, whose keys are loaded together: with several
// waves of a SIMD at different places that keeps HBM busy. A second set of keys under way while one is worked on
// costs the registers of a wave in flight, and measured slower (64 x 4096 tokens, 32 rows: stats 100 -> 110 us;
// the loads alone, with nothing worked out, take 93 us).
template <bool BF16, int STEPS, int NT>
constexpr int few_tiles() {
    const int n = BF16 ? (STEPS <= 4 ? 4 : 2) : (STEPS <= 2 ? 4 : STEPS <= 4 ? 2 : 1);
    return NT == 4 && n > 1 ? n / 2 : n;
}

// A wave's way through the keys of an item.
template <bool BF16, int STEPS, bool FULL, int U>
struct Keys {
    Frag<BF16> k[U][STEPS];
    int64_t blk[U];  // of the tiles to be loaded next
    bool ok[U];      // this lane's token is there
    int b, h, t0, end;

    __device__ __forceinline__ void ids(const AttnWeightsArgs& a, int t) {
        const int col = threadIdx.x & 15;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = t + 16 * u + col;
            blk[u] = at < end ? block_of(a, b, at) : -1;
        }
    }
    // Tiles from t on; then the block ids of the ones behind them.
    __device__ __forceinline__ void load(const AttnWeightsArgs& a, int t) {
        const int lane = threadIdx.x & 63, col = lane & 15;
        int64_t off[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = t + 16 * u + col;
            off[u] = at < end ? key_offset(a, blk[u], h, at) : -1;
            ok[u] = off[u] >= 0;
        }
        ids(a, t + 16 * U);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (t + 16 * u >= end) continue;  // uniform
            const size_t from = off[u] >= 0 ? (size_t)off[u] : 0;  // a token that is not there is masked below
#pragma unroll
            for (int i = 0; i < STEPS; ++i) k[u][i].template load<FULL>(a.k, from, i, i == STEPS - 1, a.D, lane);
        }
    }
};

// The item's wave quarter.
__device__ __forceinline__ void wave_part(const AttnWeightsArgs& a, const Sequence& s, int chunk, int& t0, int& end) {
    const int quarter = a.chunk / kWaves;  // a multiple of 16
    t0 = chunk * a.chunk + (threadIdx.x >> 6) * quarter;
    end = min(s.ctx, t0 + quarter);
}

__device__ __forceinline__ int few_items(const AttnWeightsArgs& a, int ctx, int n) {
    return n * a.group <= a.few_rows ? (ctx + a.chunk - 1) / a.chunk * a.Hkv : 0;
}

// The sum over a row of 16 lanes is row16_sum; this is the maximum.
__device__ __forceinline__ float row16_max(float v) {
    v = fmaxf(v, __int_as_float(KYRO_DPP(__float_as_int(v), 0xB1, 0xF)));   // quad_perm [1,0,3,2]
    v = fmaxf(v, __int_as_float(KYRO_DPP(__float_as_int(v), 0x4E, 0xF)));   // quad_perm [2,3,0,1]
    v = fmaxf(v, __int_as_float(KYRO_DPP(__float_as_int(v), 0x141, 0xF)));  // row_half_mirror
    return fmaxf(v, __int_as_float(KYRO_DPP(__float_as_int(v), 0x140, 0xF)));  // row_mirror
}

template <bool BF16, int STEPS, bool FULL, int NT, bool KEEP>
__global__ __launch_bounds__(kThreads) void few_stats_kernel(AttnWeightsArgs a) {
    constexpr int U = few_tiles<BF16, STEPS, NT>();
    __shared__ float2 stat[kWaves][NT * 16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = lane & 15, quad = lane >> 4;
    const auto items_of = [&](int ctx, int n) { return few_items(a, ctx, n); };
    Walk walk;
    Sequence s;
    for (int64_t item = blockIdx.x; walk.find(a, false, item, items_of, s); item += gridDim.x) {
        const int rows = s.n * a.group, rest = (int)(item - s.first);
        const int h = rest % a.Hkv, chunk = rest / a.Hkv;
        Keys<BF16, STEPS, FULL, U> keys;
        int t0, end;
        wave_part(a, s, chunk, t0, end);
        keys.b = s.b;
        keys.h = h;
        keys.end = end;
        keys.ids(a, t0);
        Frag<BF16> q[NT][STEPS];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {  // rows behind the last are zeros: their statistics are not stored
            const int r = nt * 16 + col;
            load_row<BF16, STEPS, FULL>(q[nt], a.q, r < rows ? (int64_t)query_row(a, s, h, r) * a.D : -1, a.D, lane);
        }
        float m[NT][4], l[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                m[nt][i] = kNegInf;
                l[nt][i] = 0.f;
            }
        const int whole = last_seen(a, s, 0);  // tokens up to it are seen by all rows
        float* kept = nullptr;
        if constexpr (KEEP) {
            if (item < a.kept_items) kept = a.kept + (size_t)item * a.chunk * a.kept_rows;
        }
        for (; t0 < end; t0 += 16 * U) {
            keys.load(a, t0);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float x[4][U];
                f32x4 c[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    c[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < STEPS; ++i) c[u] = Frag<BF16>::mma(q[nt][i], keys.k[u][i], c[u]);
                    const bool hide = !keys.ok[u];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float v = c[u][i] * a.scale_log2;
                        // A kept -infinity is a score that is not seen. One that is seen stays apart from it:
                        // a row that has a NaN gives it one.
                        if constexpr (KEEP) v = v == kNegInf ? -FLT_MAX : v;
                        x[i][u] = hide ? kNegInf : v;
                    }
                }
                if (t0 + 16 * U - 1 > whole) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int last = last_seen(a, s, nt * 16 + quad * 4 + i);
#pragma unroll
                        for (int u = 0; u < U; ++u) x[i][u] = t0 + 16 * u + col > last ? kNegInf : x[i][u];
                    }
                }
                if constexpr (KEEP) {
                    if (kept && nt * 16 + quad * 4 < a.kept_rows) {
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            const int at = t0 - chunk * a.chunk + 16 * u + col;
                            if (t0 + 16 * u < end)
                                *reinterpret_cast<float4*>(kept + ((size_t)(nt * 4 + quad) * a.chunk + at) * 4) =
                                    make_float4(x[0][u], x[1][u], x[2][u], x[3][u]);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) add_scores<U>(m[nt][i], l[nt][i], x[i]);
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float top = row16_max(m[nt][i]);
                float sum = row16_sum(l[nt][i] * (m[nt][i] == kNegInf ? 1.f : fast_exp2(m[nt][i] - top)));
                if (KEEP && top == -FLT_MAX) {  // no score above -infinity
                    top = kNegInf;
                    sum = sum == sum ? 0.f : sum;
                }
                if (col == 0) stat[wave][nt * 16 + quad * 4 + i] = make_float2(top, sum);
            }
        __syncthreads();
        for (int r = threadIdx.x; r < min(rows, NT * 16); r += kThreads) {
            float2 x = stat[0][r];
            for (int w = 1; w < kWaves; ++w) merge(x.x, x.y, stat[w][r].x, stat[w][r].y);
            a.part[(size_t)chunk * a.total_q * a.H + query_row(a, s, h, r)] = x;
        }
        __syncthreads();
    }
}

// The sums of items whose scores were not kept, from their keys.
template <bool BF16, int STEPS, bool FULL, int NT>
__global__ __launch_bounds__(kThreads) void few_sum_kernel(AttnWeightsArgs a) {
    constexpr int U = few_tiles<BF16, STEPS, NT>();
    __shared__ float lse[NT * 16];
    __shared__ float2 partial[kThreads];
    const int lane = threadIdx.x & 63;
    const int col = lane & 15, quad = lane >> 4;
    const auto items_of = [&](int ctx, int n) { return few_items(a, ctx, n); };
    const bool backwards = a.kept_items == 0;  // the kept ones are the first
    Walk walk;
    Sequence s;
    for (int64_t item = a.kept_items + blockIdx.x; walk.find(a, backwards, item, items_of, s); item += gridDim.x) {
        const int rows = s.n * a.group, parts = (s.ctx + a.chunk - 1) / a.chunk;
        const int rest = (int)(item - s.first);
        const int h = rest % a.Hkv, chunk = backwards ? parts - 1 - rest / a.Hkv : rest / a.Hkv;
        const int64_t row = state_row(a, s.b);
        if (row < 0) continue;
        Keys<BF16, STEPS, FULL, U> keys;
        int t0, end;
        wave_part(a, s, chunk, t0, end);
        keys.b = s.b;
        keys.h = h;
        keys.end = end;
        keys.ids(a, t0);
        Frag<BF16> q[NT][STEPS];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = nt * 16 + col;
            load_row<BF16, STEPS, FULL>(q[nt], a.q, r < rows ? (int64_t)query_row(a, s, h, r) * a.D : -1, a.D, lane);
        }
        merge_chunks<NT * 16>(a, s, h, parts, partial, lse);
        float to[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) to[nt][i] = lse[nt * 16 + quad * 4 + i];
        const int whole = last_seen(a, s, 0);
        const size_t base = ((size_t)row * a.Hkv + h) * a.max_tokens;
        for (; t0 < end; t0 += 16 * U) {
            float w[U];
#pragma unroll
            for (int u = 0; u < U; ++u) w[u] = quad == 0 ? old_weight(a, s, base, t0 + 16 * u + col, end) : 0.f;
            keys.load(a, t0);
            float sum[U];
#pragma unroll
            for (int u = 0; u < U; ++u) sum[u] = 0.f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float p[4][U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < STEPS; ++i) c = Frag<BF16>::mma(q[nt][i], keys.k[u][i], c);
#pragma unroll
                    for (int i = 0; i < 4; ++i) p[i][u] = fast_exp2(c[i] * a.scale_log2 - to[nt][i]);
                }
                if (t0 + 16 * U - 1 > whole || rows < NT * 16) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = nt * 16 + quad * 4 + i, last = r < rows ? last_seen(a, s, r) : -1;
#pragma unroll
                        for (int u = 0; u < U; ++u) p[i][u] = t0 + 16 * u + col > last ? 0.f : p[i][u];
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u) sum[u] += (p[0][u] + p[1][u]) + (p[2][u] + p[3][u]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float x = sum[u];
                x += shfl_xor_f(x, 16);
                x += shfl_xor_f(x, 32);
                const int t = t0 + 16 * u + col;
                if (quad == 0 && t < end) store_weight(a, s, base, t, w[u] + (keys.ok[u] ? x : 0.f));
            }
        }
    }
    if (a.idle == kIdleFewSum) copy_idle(a);
}

// The sums of items whose scores were kept: a thread has a token.
constexpr int kKeptRows = 32;  // most rows of a kv head that keep their scores
__global__ __launch_bounds__(kThreads) void kept_sum_kernel(AttnWeightsArgs a) {
    __shared__ float lse[kKeptRows];
    __shared__ float2 partial[kThreads];
    const auto items_of = [&](int ctx, int n) { return few_items(a, ctx, n); };
    Walk walk;
    Sequence s;
    for (int64_t item = blockIdx.x; item < a.kept_items && walk.find(a, false, item, items_of, s); item += gridDim.x) {
        const int parts = (s.ctx + a.chunk - 1) / a.chunk, rest = (int)(item - s.first);
        const int h = rest % a.Hkv, chunk = rest / a.Hkv;
        const int64_t row = state_row(a, s.b);
        if (row < 0) continue;
        const size_t base = ((size_t)row * a.Hkv + h) * a.max_tokens;
        const int end = min(s.ctx, (chunk + 1) * a.chunk);
        const float* kept = a.kept + (size_t)item * a.chunk * a.kept_rows;
        merge_chunks<kKeptRows>(a, s, h, parts, partial, lse);
        for (int t = chunk * a.chunk + threadIdx.x; t < end; t += kThreads) {
            const float4* x = reinterpret_cast<const float4*>(kept) + (t - chunk * a.chunk);
            const float w = old_weight(a, s, base, t, end);
            float sum = 0.f;
            for (int r = 0; r < a.kept_rows; r += 4) {
                const float4 v = x[(size_t)(r / 4) * a.chunk];
                // What a row does not see was kept as -infinity, and adds nothing to it even where the row
                // has a NaN. What fills up the last rows (lse infinity) adds nothing even where the token has one.
                const float p0 = ((v.x == kNegInf) | (lse[r] == -kNegInf)) ? 0.f : fast_exp2(v.x - lse[r]);
                const float p1 = ((v.y == kNegInf) | (lse[r + 1] == -kNegInf)) ? 0.f : fast_exp2(v.y - lse[r + 1]);
                const float p2 = ((v.z == kNegInf) | (lse[r + 2] == -kNegInf)) ? 0.f : fast_exp2(v.z - lse[r + 2]);
                const float p3 = ((v.w == kNegInf) | (lse[r + 3] == -kNegInf)) ? 0.f : fast_exp2(v.w - lse[r + 3]);
                sum += (p0 + p1) + (p2 + p3);
            }
            store_weight(a, s, base, t, w + sum);
        }
    }
    if (a.idle == kIdleKeptSum) copy_idle(a);
}

// ------------------------------------------------------------------- many rows (prompts)

// Both passes of a prompt are one product of a stationary operand, 16 NT vectors of which each wave holds in
// registers, with a streamed one that the four waves share through LDS, double buffered, kTile vectors at
// a time, laid out as the operands of the products.
//   stats  stationary: query rows;  streamed: a chunk's keys.    Item: (sequence, chunk, kv head, row group)
//   sum    stationary: keys;        streamed: the query rows.    Item: (sequence, run of tokens, kv head, part
//          of the rows); with several parts (few tokens, many rows) their sums are joined by join_kernel
// Whether any score of a streamed tile is hidden is decided once for the wave, and the tile is worked on
// without a branch: a branch per 16 x 16 scores kept their products and exponentials apart. On 2 x 512 rows at
// 8192 tokens, 32/8 heads of 128 (2 x 69 GFLOP), stats take 127 us and sum 101 us, 540 and 680 TFLOP/s where a
// large library product reaches 1245. With a quarter of the products sum takes 79 us, without the exponentials
// 90 us, without both 62 us: what is left is the tiles' way through LDS and the barriers.
template <bool BF16, int FRAGS, int N>
struct Staged {
    uint4 x[FRAGS][BF16 ? 1 : 2][64];  // operand f's 16-byte pieces, one a lane
    float lse[N];  // sum: of the streamed rows
    int last[N];   // sum: the last token each streamed row sees; stats: -1 for no token
    int gap;       // stats: some token of the tile is not there
};
template <bool BF16, int STEPS>
constexpr int many_tiles() { return BF16 || STEPS <= 4 ? 4 : 2; }
template <bool BF16, int STEPS>
constexpr int many_streamed() { return BF16 && STEPS <= 4 ? 64 : 32; }

template <bool BF16, int STEPS, bool FULL, bool SUM>
__global__ __launch_bounds__(kThreads) void many_kernel(AttnWeightsArgs a) {
    constexpr int NT = many_tiles<BF16, STEPS>(), kTile = many_streamed<BF16, STEPS>();
    constexpr int kSub = kTile / 16, kHold = kWaves * NT * 16;
    constexpr int kLoads = (kSub * STEPS + kWaves - 1) / kWaves;  // operands of a tile, for each wave
    // Two arrays, not one of two: what is loaded into one is then known not to touch the other.
    __shared__ Staged<BF16, kSub * STEPS, kTile> tile0, tile1;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = lane & 15, quad = lane >> 4;
    const auto items_of = [&](int ctx, int n) {
        const int rows = n * a.group;
        if (rows <= a.few_rows) return 0;
        return SUM ? (ctx + kHold - 1) / kHold * a.Hkv * a.row_parts
                   : (ctx + a.chunk - 1) / a.chunk * a.Hkv * ((rows + kHold - 1) / kHold);
    };
    Walk walk;
    Sequence s;
    for (int64_t item = blockIdx.x; walk.find(a, SUM, item, items_of, s); item += gridDim.x) {
        const int rows = s.n * a.group, old = s.ctx - s.n;
        int rest = (int)(item - s.first), row0 = 0, h, chunk = 0, run0 = 0, part = 0;
        int64_t row = 0;
        if constexpr (SUM) {
            part = rest % a.row_parts;
            rest /= a.row_parts;
            h = rest % a.Hkv;
            run0 = ((s.ctx + kHold - 1) / kHold - 1 - rest / a.Hkv) * kHold;
            if (a.row_parts == 1) {
                row = state_row(a, s.b);
                if (row < 0) continue;
            }
        } else {
            const int groups = (rows + kHold - 1) / kHold;
            // The last rows see the most tokens: their groups first.
            row0 = (groups - 1 - rest % groups) * kHold;
            rest /= groups;
            h = rest % a.Hkv;
            chunk = rest / a.Hkv;
        }
        const int hold0 = (SUM ? run0 : row0) + wave * NT * 16;  // the wave's first stationary vector
        Frag<BF16> x[NT][STEPS];
        bool there[NT];
        int limit[NT];  // stats: the last token the lane's row sees
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int v = hold0 + nt * 16 + col;
            int64_t off;
            if constexpr (SUM) {
                off = v < s.ctx ? key_offset(a, block_of(a, s.b, v), h, v) : -1;
                limit[nt] = 0;
            } else {
                off = v < rows ? (int64_t)query_row(a, s, h, v) * a.D : -1;
                limit[nt] = v < rows ? last_seen(a, s, v) : -1;
            }
            there[nt] = off >= 0;
            load_row<BF16, STEPS, FULL>(x[nt], SUM ? a.k : a.q, off, a.D, lane);
        }
        // Streamed vectors [from, to): rows that see something of the run, or the chunk's tokens that the
        // group's last row sees.
        int from, to;
        if constexpr (SUM) {
            from = a.causal ? max(0, run0 - old) * a.group / kTile * kTile : 0;
            const int per = ((rows - from + kTile - 1) / kTile + a.row_parts - 1) / a.row_parts * kTile;
            from += part * per;
            to = min(rows, from + per);
        } else {
            from = chunk * a.chunk;
            to = min(min(s.ctx, from + a.chunk), last_seen(a, s, min(rows, row0 + kHold) - 1) + 1);
        }
        // A tile's vectors: whole rows straight into LDS (FULL), where they land while the tile before is worked on,
        // others by way of the registers, which put zeros behind their last element. Vectors that are not there
        // repeat element 0 or the last row: their scores are hidden.
        constexpr int kHeld = FULL ? 1 : kLoads;
        Frag<BF16> buf[kHeld];
        float buf_lse = 0.f;
        int buf_last = 0;
        int64_t blk[kLoads], blk_last = 0;  // stats: the block ids of the tile to be fetched next
        const auto ids = [&](int v0) {
            if constexpr (!SUM) {
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    const int v = v0 + (i * kWaves + wave) / STEPS * 16 + col;
                    blk[i] = v < to ? block_of(a, s.b, v) : 0;
                }
                const int v = v0 + threadIdx.x;
                if (threadIdx.x < kTile) blk_last = v < to ? block_of(a, s.b, v) : 0;
            }
        };
        const auto fetch = [&](Staged<BF16, kSub * STEPS, kTile>& into, int v0) {
            int64_t off[kLoads];
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int v = v0 + (i * kWaves + wave) / STEPS * 16 + col;
                if constexpr (SUM) off[i] = (int64_t)query_row(a, s, h, min(v, to - 1)) * a.D;
                else off[i] = v < to ? max((int64_t)0, key_offset(a, blk[i], h, v)) : 0;
            }
            if (threadIdx.x < kTile) {
                const int v = v0 + threadIdx.x;
                if constexpr (SUM) {
                    buf_lse = v < to ? a.lse[query_row(a, s, h, v)] : -kNegInf;
                    buf_last = v < to ? last_seen(a, s, v) : -1;
                } else {
                    buf_last = v < to && blk_last >= 0 && blk_last < a.num_blocks ? v : -1;
                }
            }
            ids(v0 + kTile);
            constexpr int kSize = BF16 ? 2 : 4;
            const char* base = reinterpret_cast<const char*>(SUM ? a.q : a.k);
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int f = i * kWaves + wave;
                if (kSub * STEPS % kWaves != 0 && f >= kSub * STEPS) break;
                if constexpr (FULL) {
#pragma unroll
                    for (int p = 0; p < (BF16 ? 1 : 2); ++p) {
                        const size_t at = (size_t)off[i] + Frag<BF16>::piece(f % STEPS, f % STEPS == STEPS - 1, p, lane);
                        __builtin_amdgcn_global_load_lds(
                            (const __attribute__((address_space(1))) void*)(base + at * kSize),
                            (__attribute__((address_space(3))) void*)&into.x[f][p][0], 16, 0, 0);
                    }
                } else {
                    buf[i].template load<FULL>(base, (size_t)off[i], f % STEPS, f % STEPS == STEPS - 1, a.D, lane);
                }
            }
        };
        // Ends a fetch: after the barrier behind it the tile may be read.
        const auto stage = [&](Staged<BF16, kSub * STEPS, kTile>& into) {
            if constexpr (!FULL) {
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    const int f = i * kWaves + wave;
                    if (kSub * STEPS % kWaves == 0 || f < kSub * STEPS) buf[i].put(into.x[f], lane);
                }
            }
            if (threadIdx.x < kTile) {
                into.lse[threadIdx.x] = buf_lse;
                into.last[threadIdx.x] = buf_last;
                if (!SUM) {
                    const bool any = __ballot(buf_last < 0) != 0;
                    if (threadIdx.x == 0) into.gap = any;
                }
            }
            if constexpr (FULL) __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's loads have landed
            __syncthreads();
        };
        float m[NT], l[NT];  // stats: running maximum and sum; sum: l is the token's weight
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt] = kNegInf;
            l[nt] = 0.f;
        }
        __syncthreads();  // the item before has read its tiles
        if (from < to) {
            ids(from);
            fetch(tile0, from);
            stage(tile0);
        }
        const bool mine = hold0 < (SUM ? s.ctx : rows);
        const int whole = SUM ? 0 : last_seen(a, s, min(hold0, rows - 1));  // seen by all of the wave's rows
        // A streamed tile, two 16-vector parts at a time. EDGE: some of its scores are hidden.
        const auto product = [&](f32x4 (&c)[2][NT], const Staged<BF16, kSub * STEPS, kTile>& in, int sub) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) c[j][nt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    Frag<BF16> y;
                    y.get(in.x[(sub + j) * STEPS + i], lane);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) c[j][nt] = Frag<BF16>::mma(y, x[nt][i], c[j][nt]);
                }
            }
        };
        const auto scores = [&](auto edge, const f32x4 (&c)[2][NT], const Staged<BF16, kSub * STEPS, kTile>& in, int sub,
                                int v0) {
            constexpr bool EDGE = decltype(edge)::value;
            float set[2][4];
            int see[2][4];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (SUM) set[j][i] = in.lse[(sub + j) * 16 + quad * 4 + i];
                    if (EDGE) see[j][i] = in.last[(sub + j) * 16 + quad * 4 + i];
                }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                if constexpr (SUM) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float p[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            p[i] = fast_exp2(c[j][nt][i] * a.scale_log2 - set[j][i]);
                            if (EDGE) p[i] = hold0 + nt * 16 + col > see[j][i] ? 0.f : p[i];
                        }
                        l[nt] += (p[0] + p[1]) + (p[2] + p[3]);
                    }
                } else {
                    float p[8];
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            p[4 * j + i] = c[j][nt][i];
                            if (EDGE) {
                                const bool hidden = (see[j][i] < 0) | (v0 + (sub + j) * 16 + quad * 4 + i > limit[nt]);
                                p[4 * j + i] = hidden ? kNegInf : p[4 * j + i];
                            }
                        }
                    add_products<8>(m[nt], l[nt], p, a.scale_log2);
                }
            }
        };
        const auto work = [&](auto edge, const Staged<BF16, kSub * STEPS, kTile>& in, int v0) {
#pragma unroll
            for (int sub = 0; sub < kSub; sub += 2) {
                f32x4 c[2][NT];
                product(c, in, sub);
                scores(edge, c, in, sub, v0);
            }
        };
        // sum: the wave's last token against what the tile's first row sees.
        const auto turn = [&](Staged<BF16, kSub * STEPS, kTile>& in, Staged<BF16, kSub * STEPS, kTile>& next, int v0) {
            const bool more = v0 + kTile < to;
            if (more) fetch(next, v0 + kTile);
            if (mine) {
                const bool edge = v0 + kTile > to ||
                                  (SUM ? hold0 + NT * 16 - 1 > __builtin_amdgcn_readfirstlane(in.last[0])
                                       : v0 + kTile - 1 > whole || __builtin_amdgcn_readfirstlane(in.gap) != 0);
                if (edge) work(std::true_type{}, in, v0);
                else work(std::false_type{}, in, v0);
            }
            if (more) stage(next);
        };
        for (int v0 = from; v0 < to; v0 += 2 * kTile) {
            turn(tile0, tile1, v0);
            if (v0 + kTile < to) turn(tile1, tile0, v0 + kTile);
        }
        if constexpr (SUM) {
            const size_t base = ((size_t)row * a.Hkv + h) * a.max_tokens;
            float* parts = a.row_sums + (((size_t)part * a.B + s.b) * a.Hkv + h) * a.run_tokens;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int t = hold0 + nt * 16 + col;
                float w = l[nt];
                w += shfl_xor_f(w, 16);
                w += shfl_xor_f(w, 32);
                w = there[nt] ? w : 0.f;
                if (quad == 0 && t < s.ctx) {
                    if (a.row_parts == 1) store_weight(a, s, base, t, old_weight(a, s, base, t, s.ctx) + w);
                    else parts[t] = w;
                }
            }
        } else {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int j = 16; j <= 32; j <<= 1) merge(m[nt], l[nt], shfl_xor_f(m[nt], j), shfl_xor_f(l[nt], j));
                const int r = hold0 + nt * 16 + col;
                if (quad == 0 && r < rows)
                    a.part[(size_t)chunk * a.total_q * a.H + query_row(a, s, h, r)] = make_float2(m[nt], l[nt]);
            }
        }
    }
}

// Adds up the parts of the many-row sums, in their order. Item: (sequence, run of kThreads tokens, kv head).
__global__ __launch_bounds__(kThreads) void join_kernel(AttnWeightsArgs a) {
    const auto items_of = [&](int ctx, int n) {
        return n * a.group <= a.few_rows ? 0 : (ctx + kThreads - 1) / kThreads * a.Hkv;
    };
    Walk walk;
    Sequence s;
    for (int64_t item = blockIdx.x; walk.find(a, false, item, items_of, s); item += gridDim.x) {
        const int rest = (int)(item - s.first), h = rest % a.Hkv, t = rest / a.Hkv * kThreads + threadIdx.x;
        const int64_t row = state_row(a, s.b);
        if (row < 0 || t >= s.ctx) continue;
        const size_t base = ((size_t)row * a.Hkv + h) * a.max_tokens;
        const float* parts = a.row_sums + ((size_t)s.b * a.Hkv + h) * a.run_tokens + t;
        float w = 0.f;
        for (int i = 0; i < a.row_parts; ++i) w += parts[(size_t)i * a.B * a.Hkv * a.run_tokens];
        store_weight(a, s, base, t, old_weight(a, s, base, t, s.ctx) + w);
    }
}

// The rows' statistics merged over their chunks, one thread a (row, head).
__device__ __forceinline__ void merge_row(const AttnWeightsArgs& a, int64_t i, int64_t all) {
    const int r = (int)(i / a.H);
    // The row's sequence tells how many chunks there are; a row of none, or of one left out, has no
    // statistics.
    int lo = 0, hi = a.B;  // the number of q_start[1..] that are <= r
    if (a.q_start) {
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (a.q_start[mid + 1] <= r) lo = mid + 1;
            else hi = mid;
        }
    } else {
        lo = r;
    }
    if (lo >= a.B) return;
    const int64_t ctx = a.ctx_lens[lo];
    if (ctx < 0 || ctx > a.cap) return;
    const int parts = (int)((ctx + a.chunk - 1) / a.chunk);
    float m = kNegInf, l = 0.f;
    for (int c = 0; c < parts; ++c) {
        const float2 x = a.part[c * all + i];
        merge(m, l, x.x, x.y);
    }
    a.lse[i] = log_sum(m, l);
}
__global__ __launch_bounds__(kThreads) void merge_kernel(AttnWeightsArgs a) {
    const int64_t all = (int64_t)a.total_q * a.H, i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i < all) merge_row(a, i, all);
    if (a.idle == kIdleMerge) copy_idle(a);
}

template <bool BF16, int STEPS, bool FULL>
void launch_steps(const AttnWeightsArgs& a, hipStream_t stream) {
    if (a.few_grid) {
        const bool rest = a.few_items_most > a.kept_items;  // there may be items whose scores are not kept
        if (a.few_rows == 16) {
            few_stats_kernel<BF16, STEPS, FULL, 1, true><<<a.few_grid, kThreads, 0, stream>>>(a);
            if (rest) few_sum_kernel<BF16, STEPS, FULL, 1><<<a.few_grid, kThreads, 0, stream>>>(a);
        } else if (a.few_rows == 32) {
            if (a.kept_items) few_stats_kernel<BF16, STEPS, FULL, 2, true><<<a.few_grid, kThreads, 0, stream>>>(a);
            else few_stats_kernel<BF16, STEPS, FULL, 2, false><<<a.few_grid, kThreads, 0, stream>>>(a);
            if (rest) few_sum_kernel<BF16, STEPS, FULL, 2><<<a.few_grid, kThreads, 0, stream>>>(a);
        } else {
            constexpr int NT = BF16 || STEPS <= 4 ? 4 : 2;
            few_stats_kernel<BF16, STEPS, FULL, NT, false><<<a.few_grid, kThreads, 0, stream>>>(a);
            few_sum_kernel<BF16, STEPS, FULL, NT><<<a.few_grid, kThreads, 0, stream>>>(a);
        }
        if (a.kept_items) kept_sum_kernel<<<a.few_grid, kThreads, 0, stream>>>(a);
    }
    if (a.many_stat_grid) {
        many_kernel<BF16, STEPS, FULL, false><<<a.many_stat_grid, kThreads, 0, stream>>>(a);
        merge_kernel<<<(unsigned)(((int64_t)a.total_q * a.H + kThreads - 1) / kThreads), kThreads, 0, stream>>>(a);
        many_kernel<BF16, STEPS, FULL, true><<<a.many_sum_grid, kThreads, 0, stream>>>(a);
        if (a.row_parts > 1) join_kernel<<<a.many_sum_grid, kThreads, 0, stream>>>(a);
    }
}

template <bool BF16>
void launch_type(const AttnWeightsArgs& a, hipStream_t stream) {
    switch (a.D) {
        case 32: return launch_steps<BF16, 1, true>(a, stream);
        case 64: return launch_steps<BF16, 2, true>(a, stream);
        case 96: return launch_steps<BF16, 3, true>(a, stream);
        case 128: return launch_steps<BF16, 4, true>(a, stream);
        case 192: return launch_steps<BF16, 6, true>(a, stream);
        case 256: return launch_steps<BF16, 8, true>(a, stream);
        default: break;
    }
    // Others take the next of three sizes, with zeros behind their last element: fewer kernels to build, not the
    // fastest (2 x 512 rows at 8192 tokens, 32/8 heads: 330 us at 136, where 192 takes 264; 198 at 72, 169 at 96).
    if (a.D < 64) return launch_steps<BF16, 2, false>(a, stream);
    if (a.D < 128) return launch_steps<BF16, 4, false>(a, stream);
    launch_steps<BF16, 8, false>(a, stream);
}

}  // namespace

#if KYRO_WEIGHTS_F32
void launch_attn_weights_f32(const AttnWeightsArgs& a, hipStream_t stream) { launch_type<false>(a, stream); }
#else
int attn_weights_few_rows(bool bf16, int D) { return bf16 || D <= 128 ? 64 : 32; }
int attn_weights_many_hold(bool bf16, int D) { return bf16 || D <= 128 ? 256 : 128; }

hipError_t launch_attn_weights(const AttnWeightsArgs& a, hipStream_t stream) {
    if (a.B == 0) return hipSuccess;
    if (a.total_q == 0) {  // no row: the merge of none, which takes the sequences' weights along
        if (a.idle) merge_kernel<<<(unsigned)(a.B < 256 ? 256 : 2048), kThreads, 0, stream>>>(a);
    } else if (a.bf16) {
        launch_type<true>(a, stream);
    } else {
        launch_attn_weights_f32(a, stream);
    }
    return hipGetLastError();
}
#endif

}  // namespace kyro
