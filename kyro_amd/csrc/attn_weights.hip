// Accumulated attention weight of cached tokens (gfx950): for each kv head and cached token t,
//     w[t] += sum over the step's query rows r of that head's group of  exp(s[r,t] - m[r]) / l[r],
//     s[r,t] = scale q_r . k_t over the tokens r sees,  m[r] = max_t s,  l[r] = sum_t exp(s - m).
//
// The sum over rows needs every row's m and l first, and keeping the scores costs 4 bytes a row and token
// each way against 2 D bytes to read the token's key again. Two passes over K:
//   stats   m and l of each row over a chunk of tokens, one running maximum and sum per lane;
//   sum     a wave holds the keys of its tokens in registers, takes the rows 32 at a time from LDS with
//           their m + log l merged over the chunks, and adds up exp2(s - that) per token.
// One wave owns a token's sum and adds rows in order: no atomics, the same result every time.
//
// Both products run on MFMA with the operands' roles chosen so that what is reduced lies in one lane: the
// 16 x 16 result has the first operand's index in the lane's four registers and the second's in the lane,
// so stats takes (K, Q) - a lane has one row and four tokens - and sum takes (Q, K). Both operands of a
// 16x16x32 product hold 8 elements of row lane % 16 from element 8 (lane / 16): keys and queries go from
// memory straight into them, 16 bytes a lane, whatever the block size. The f32 caches take 16x16x4 products
// on 4-element pieces, the same pieces for both operands.
#include "common.hpp"
#include "kernels.hpp"

namespace kyro {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

// 32 elements of 16 rows as one operand: element e of lane l is row l % 16's element 8 (l / 16) + e (bf16)
// or 4 (l / 16) + e % 4 + 16 (e / 4) (f32).
template <bool BF16>
struct Frag;
template <>
struct Frag<true> {
    bf16x8 x;
    __device__ __forceinline__ void load(const void* base, size_t row, int d, int D, int lane) {
        const int at = d + 8 * (lane >> 4);
        uint4 u = make_uint4(0, 0, 0, 0);
        if (at < D) u = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(base) + row + at);
        x = __builtin_bit_cast(bf16x8, u);
    }
    __device__ __forceinline__ void zero() { x = __builtin_bit_cast(bf16x8, make_uint4(0, 0, 0, 0)); }
    static __device__ __forceinline__ f32x4 mma(const Frag& a, const Frag& b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.x, b.x, c, 0, 0, 0);
    }
};
template <>
struct Frag<false> {
    f32x4 x[2];
    __device__ __forceinline__ void load(const void* base, size_t row, int d, int D, int lane) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int at = d + 16 * i + 4 * (lane >> 4);
            x[i] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (at < D) x[i] = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(base) + row + at);
        }
    }
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
// each counted from its own length. Items of a workgroup rise, so the walk goes on where it was.
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

    // Items of a sequence: PER_ITEM(ctx, n). Wave-uniform; false behind the last item.
    template <typename F>
    __device__ __forceinline__ bool find(const AttnWeightsArgs& a, int64_t item, F per_sequence, Sequence& s) {
        const int lane = threadIdx.x & 63;
        while (item >= base + total) {
            base += total;
            strip += 64;
            if (strip >= a.B) return false;
            const int b = strip + lane;
            int count = 0;
            n = ctx = 0;
            if (b < a.B) {
                int r0 = b, r1 = b + 1;
                if (a.q_start) {
                    r0 = a.q_start[b];
                    r1 = a.q_start[b + 1];
                }
                const int64_t c = a.ctx_lens[b];
                int bad = 0;
                if (r0 < 0 || r1 < r0 || r1 > a.total_q || r1 - r0 > a.max_q_len) bad |= ERR_Q_LAYOUT;
                else if (c < r1 - r0 || c > a.cap) bad |= ERR_CTX_LEN;
                if (bad) {
                    latch_error(a.err, bad);
                } else if (r1 > r0) {
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
        s.b = strip + l;
        s.q0 = __builtin_amdgcn_readlane(q0, l);
        s.n = __builtin_amdgcn_readlane(n, l);
        s.ctx = __builtin_amdgcn_readlane(ctx, l);
        s.first = base + (l ? __builtin_amdgcn_readlane(incl, l - 1) : 0);
        return true;
    }
};

// Element offset of a cached token's key, or -1 for a bad block.
__device__ __forceinline__ int64_t key_offset(const AttnWeightsArgs& a, int b, int h, int t) {
    const int page = a.bs_shift >= 0 ? t >> a.bs_shift : t / a.bs;
    const int64_t blk = a.table[(size_t)b * a.max_blocks + page];
    if (blk < 0 || blk >= a.num_blocks) {
        latch_error(a.err, ERR_BLOCK_ID);
        return -1;
    }
    return ((blk * a.Hkv + h) * a.bs + (t - page * a.bs)) * a.D;
}

// Element offset of row r (of a kv head's n * group rows, row by row) in the query.
__device__ __forceinline__ size_t query_row(const AttnWeightsArgs& a, const Sequence& s, int h, int r) {
    const int j = r / a.group;
    return (size_t)(s.q0 + j) * a.H + (size_t)h * a.group + (r - j * a.group);
}

// The last token that row r sees.
__device__ __forceinline__ int last_seen(const AttnWeightsArgs& a, const Sequence& s, int r) {
    return a.causal ? s.ctx - s.n + r / a.group : s.ctx - 1;
}

// The running (max, sum) of two sets of scores, in base 2. The sum that goes with a maximum of -infinity is
// 0, or NaN where a score was: that has to reach the result.
__device__ __forceinline__ void merge(float& m, float& l, float m2, float l2) {
    const float top = fmaxf(m, m2);
    l = l * (m == kNegInf ? 1.f : fast_exp2(m - top)) + l2 * (m2 == kNegInf ? 1.f : fast_exp2(m2 - top));
    m = top;
}

// Item: (sequence, chunk of tokens, kv head, group of 16 NT rows). Each wave takes every fourth tile of 16
// tokens.
template <bool BF16, int STEPS, int NT>
__global__ __launch_bounds__(kThreads) void weights_stats_kernel(AttnWeightsArgs a) {
    __shared__ float2 stat[kWaves][NT * 16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = lane & 15, quad = lane >> 4;
    const auto items_of = [&](int ctx, int n) {
        return (ctx + a.chunk - 1) / a.chunk * a.Hkv * ((n * a.group + NT * 16 - 1) / (NT * 16));
    };
    Walk walk;
    Sequence s;
    for (int64_t item = blockIdx.x; walk.find(a, item, items_of, s); item += gridDim.x) {
        const int rows = s.n * a.group, groups = (rows + NT * 16 - 1) / (NT * 16);
        int rest = (int)(item - s.first);
        const int row0 = rest % groups * (NT * 16);
        rest /= groups;
        const int h = rest % a.Hkv, chunk = rest / a.Hkv;
        const int end = min(s.ctx, (chunk + 1) * a.chunk);
        Frag<BF16> q[NT][STEPS];
        int last[NT];
        float m[NT], l[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = row0 + nt * 16 + col;
            const bool in = r < rows;
            const size_t at = in ? query_row(a, s, h, r) * a.D : 0;
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                if (in) q[nt][i].load(a.q, at, 32 * i, a.D, lane);
                else q[nt][i].zero();
            }
            last[nt] = in ? min(last_seen(a, s, r), end - 1) : -1;
            m[nt] = kNegInf;
            l[nt] = 0.f;
        }
        // Tiles wholly behind every row's last token need no look.
        const int seen = min(end, last_seen(a, s, min(rows, row0 + NT * 16) - 1) + 1);
        const int whole = last_seen(a, s, row0);  // tokens up to it are seen by all rows
        for (int t0 = chunk * a.chunk + wave * 16; t0 < seen; t0 += kWaves * 16) {
            const int t = t0 + col;
            const int64_t off = t < end ? key_offset(a, s.b, h, t) : -1;
            Frag<BF16> k[STEPS];
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                if (off >= 0) k[i].load(a.k, (size_t)off, 32 * i, a.D, lane);
                else k[i].zero();
            }
            const bool bad = __ballot(t < end && off < 0) != 0;
            const unsigned long long gone = bad ? __ballot(off < 0) : 0;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < STEPS; ++i) c = Frag<BF16>::mma(k[i], q[nt][i], c);
                float x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = c[i] * a.scale_log2;
                if (t0 + 15 > whole || t0 + 16 > end || bad || row0 + NT * 16 > rows) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const bool hidden = (t0 + quad * 4 + i > last[nt]) | ((gone >> (quad * 4 + i)) & 1);
                        x[i] = hidden ? kNegInf : x[i];
                    }
                }
                const float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), m[nt]);
                const float ref = top == kNegInf ? 0.f : top;
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) sum += fast_exp2(x[i] - ref);
                l[nt] = l[nt] * fast_exp2(m[nt] - ref) + sum;
                m[nt] = top;
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int x = 16; x <= 32; x <<= 1) merge(m[nt], l[nt], shfl_xor_f(m[nt], x), shfl_xor_f(l[nt], x));
            if (quad == 0) stat[wave][nt * 16 + col] = make_float2(m[nt], l[nt]);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < NT * 16; i += kThreads) {
            const int r = row0 + i;
            if (r < rows) {
                float2 x = stat[0][i];
                for (int w = 1; w < kWaves; ++w) merge(x.x, x.y, stat[w][i].x, stat[w][i].y);
                a.part[(size_t)chunk * a.total_q * a.H + query_row(a, s, h, r)] = x;
            }
        }
        __syncthreads();
    }
}

// Item: (sequence, run of 4 x 16 NT tokens, kv head).
template <bool BF16, int STEPS, int NT>
__global__ __launch_bounds__(kThreads) void weights_sum_kernel(AttnWeightsArgs a) {
    __shared__ Frag<BF16> qs[kWeightRows / 16][STEPS][64];
    __shared__ float lse[kWeightRows];
    __shared__ int last[kWeightRows];  // the last token each staged row sees; -1 behind the last row
    __shared__ float2 partial[kThreads];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = lane & 15, quad = lane >> 4;
    constexpr int kRun = kWaves * NT * 16;
    const auto items_of = [&](int ctx, int) { return (ctx + kRun - 1) / kRun * a.Hkv; };
    Walk walk;
    Sequence s;
    for (int64_t item = blockIdx.x; walk.find(a, item, items_of, s); item += gridDim.x) {
        const int rest = (int)(item - s.first);
        const int h = rest % a.Hkv, run0 = rest / a.Hkv * kRun;
        const int rows = s.n * a.group, old = s.ctx - s.n;
        int64_t row = s.b;
        if (a.state_rows) {
            row = a.state_rows[s.b];
            int bad = row < 0 || row >= a.num_state_rows;
            for (int i = threadIdx.x; i < a.B; i += kThreads)
                if (i != s.b && a.state_rows[i] == (int)row) bad = 1;
            if (__syncthreads_or(bad)) {
                if (threadIdx.x == 0) latch_error(a.err, ERR_STATE_ROW);
                continue;
            }
        }
        Frag<BF16> k[NT][STEPS];
        float sum[NT];
        bool there[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int t = run0 + (wave * NT + nt) * 16 + col;
            const int64_t off = t < s.ctx ? key_offset(a, s.b, h, t) : -1;
            there[nt] = off >= 0;
            sum[nt] = 0.f;
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                if (off >= 0) k[nt][i].load(a.k, (size_t)off, 32 * i, a.D, lane);
                else k[nt][i].zero();
            }
        }
        const int parts = (s.ctx + a.chunk - 1) / a.chunk;
        // Rows whose last token lies before the run see nothing of it.
        int r0 = a.causal ? max(0, run0 - old) * a.group / kWeightRows * kWeightRows : 0;
        for (; r0 < rows; r0 += kWeightRows) {
            __syncthreads();
            for (int f = wave; f < kWeightRows / 16 * STEPS; f += kWaves) {
                const int tile = f / STEPS, i = f % STEPS, r = r0 + tile * 16 + col;
                Frag<BF16> x;
                if (r < rows) x.load(a.q, query_row(a, s, h, r) * a.D, 32 * i, a.D, lane);
                else x.zero();
                qs[tile][i][lane] = x;
            }
            {
                const int r = r0 + (threadIdx.x & (kWeightRows - 1));
                float m = kNegInf, l = 0.f;
                if (r < rows) {
                    const float2* p = a.part + query_row(a, s, h, r);
                    for (int c = threadIdx.x / kWeightRows; c < parts; c += kThreads / kWeightRows) {
                        const float2 x = p[(size_t)c * a.total_q * a.H];
                        merge(m, l, x.x, x.y);
                    }
                }
                partial[threadIdx.x] = make_float2(m, l);
            }
            __syncthreads();
            if (threadIdx.x < kWeightRows) {
                float2 x = partial[threadIdx.x];
                for (int i = 1; i < kThreads / kWeightRows; ++i)
                    merge(x.x, x.y, partial[i * kWeightRows + threadIdx.x].x, partial[i * kWeightRows + threadIdx.x].y);
                // A row that sees nothing adds exp2(s - inf) = 0.
                const int r = r0 + threadIdx.x;
                last[threadIdx.x] = r < rows ? last_seen(a, s, r) : -1;
                lse[threadIdx.x] = x.x == kNegInf && x.y == 0.f ? -kNegInf : x.x + __builtin_amdgcn_logf(x.y);
            }
            __syncthreads();
#pragma unroll
            for (int tile = 0; tile < kWeightRows / 16; ++tile) {
                const int rt = r0 + tile * 16;
                if (rt >= rows) break;
                float to[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) to[i] = lse[tile * 16 + quad * 4 + i];
                const int first_last = last_seen(a, s, rt);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < STEPS; ++i) c = Frag<BF16>::mma(qs[tile][i][lane], k[nt][i], c);
                    const int t = run0 + (wave * NT + nt) * 16 + col;
                    float p[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) p[i] = fast_exp2(c[i] * a.scale_log2 - to[i]);
                    if (run0 + (wave * NT + nt) * 16 + 15 > first_last || rt + 16 > rows) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) p[i] = t > last[tile * 16 + quad * 4 + i] ? 0.f : p[i];
                    }
                    sum[nt] += (p[0] + p[1]) + (p[2] + p[3]);
                }
            }
        }
        const size_t base = ((size_t)row * a.Hkv + h) * a.max_tokens;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int t = run0 + (wave * NT + nt) * 16 + col;
            float x = sum[nt];
            x += shfl_xor_f(x, 16);
            x += shfl_xor_f(x, 32);
            if (quad == 0 && t < s.ctx) {
                if (!there[nt]) x = 0.f;
                const bool fresh = t >= old;
                a.out_w[base + t] = fresh ? x : a.w[base + t] + x;
                if (fresh) a.positions[base + t] = a.row_pos ? (int32_t)a.row_pos[s.q0 + t - old] : t;
            }
        }
        __syncthreads();
    }
}

template <bool BF16, int STEPS>
void launch_steps(const AttnWeightsArgs& a, hipStream_t stream) {
    if (a.tiles == 1) weights_stats_kernel<BF16, STEPS, 1><<<a.stat_grid, kThreads, 0, stream>>>(a);
    else weights_stats_kernel<BF16, STEPS, 2><<<a.stat_grid, kThreads, 0, stream>>>(a);
    constexpr int kMany = BF16 || STEPS <= 4 ? 4 : 2;
    if (a.sum_tokens == 16) weights_sum_kernel<BF16, STEPS, 1><<<a.sum_grid, kThreads, 0, stream>>>(a);
    else weights_sum_kernel<BF16, STEPS, kMany><<<a.sum_grid, kThreads, 0, stream>>>(a);
}

template <bool BF16>
void launch_type(const AttnWeightsArgs& a, hipStream_t stream) {
    switch ((a.D + 31) / 32) {
        case 1: return launch_steps<BF16, 1>(a, stream);
        case 2: return launch_steps<BF16, 2>(a, stream);
        case 3: return launch_steps<BF16, 3>(a, stream);
        case 4: return launch_steps<BF16, 4>(a, stream);
        case 5:
        case 6: return launch_steps<BF16, 6>(a, stream);
        default: return launch_steps<BF16, 8>(a, stream);
    }
}

}  // namespace

hipError_t launch_attn_weights(const AttnWeightsArgs& a, hipStream_t stream) {
    if (a.B == 0 || a.total_q == 0) return hipSuccess;
    if (a.bf16) launch_type<true>(a, stream);
    else launch_type<false>(a, stream);
    return hipGetLastError();
}

}  // namespace kyro
