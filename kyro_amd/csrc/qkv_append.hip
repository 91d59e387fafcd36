// Head norms, position rotation and the paged K/V write of a step's new rows in one pass (gfx950).
//
// The reference's attention layer rotates its projected queries and keys (RotaryEmbedding,
// src/model/layers.rs:21-62, called in src/model/llama.rs:62-84) and then appends keys and values to the
// cache (src/model/kv_cache.rs:49-75). Here one launch reads the projection's output once and writes
// the query that attention reads and the cache slots. For a head row x of D elements:
//     n = x * (w + offset) / sqrt(mean(x^2) + eps)                           (optional, queries and keys)
//     y[i] = n[i] cos_i - n[i'] sin_i,  y[i'] = n[i'] cos_i + n[i] sin_i     (the first R elements)
// with i' = i + R/2 (halves) or the pairs (2i, 2i + 1) (interleaved). Everything is held in 32 bits and
// rounded once, on the store: a rounding between norm and rotation would add half a step of bf16 to
// every element for nothing.
//
// HBM-bound: each element is read once and written once, cos and sin (4 R bytes a row) come from L2.
// Layout: one wave takes 64 / LP head rows of one packed row, LP lanes each; a lane owns two chunks of E
// elements whose pairs lie in the same two chunks, so the rotation needs no exchange between lanes and
// the mean square is the only reduction (log2(LP) shuffles). A wave's row is uniform: its sequence
// (64-ary search of q_start), context length, block id and position are scalar work while the row's own
// loads, issued first, are under way.
#include "common.hpp"
#include "kernels.hpp"

namespace kyro {
namespace {

constexpr int kThreads = 256;

template <bool BF16, int E>
struct Chunk {
    float f[E];
    // The bits as loaded: a value row of the cache's own type is copied as it is, NaN payloads and all.
    uint32_t raw[BF16 ? E / 2 : 1];

    __device__ __forceinline__ void load(const void* base, size_t off) {
        if constexpr (BF16) {
            const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + off;
            if constexpr (E == 8) *reinterpret_cast<uint4*>(raw) = *reinterpret_cast<const uint4*>(p);
            else if constexpr (E == 4) *reinterpret_cast<uint2*>(raw) = *reinterpret_cast<const uint2*>(p);
            else raw[0] = *reinterpret_cast<const uint32_t*>(p);
        } else {
            load_floats<E>(reinterpret_cast<const float*>(base) + off, f);
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < E; ++i) f[i] = 0.f;
#pragma unroll
        for (int i = 0; i < (BF16 ? E / 2 : 1); ++i) raw[i] = 0;
    }
    __device__ __forceinline__ void widen() {
        if constexpr (BF16) {
#pragma unroll
            for (int i = 0; i < E / 2; ++i) {
                f[2 * i] = bf16_lo(raw[i]);
                f[2 * i + 1] = bf16_hi(raw[i]);
            }
        }
    }
    template <int N>
    static __device__ __forceinline__ void load_floats(const float* p, float* f) {
        if constexpr (N >= 4) {
#pragma unroll
            for (int i = 0; i < N / 4; ++i)
                *reinterpret_cast<float4*>(f + 4 * i) = reinterpret_cast<const float4*>(p)[i];
        } else if constexpr (N == 2) {
            *reinterpret_cast<float2*>(f) = *reinterpret_cast<const float2*>(p);
        } else {
            f[0] = p[0];
        }
    }
};

template <bool BF16, int E>
__device__ __forceinline__ void store_chunk(void* base, size_t off, const float* f) {
    if constexpr (BF16) {
        uint16_t* p = reinterpret_cast<uint16_t*>(base) + off;
        uint32_t w[E / 2];
#pragma unroll
        for (int i = 0; i < E / 2; ++i) w[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
        if constexpr (E == 8) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        else if constexpr (E == 4) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t*>(p) = w[0];
    } else {
        float* p = reinterpret_cast<float*>(base) + off;
        if constexpr (E >= 4) {
#pragma unroll
            for (int i = 0; i < E / 4; ++i)
                reinterpret_cast<float4*>(p)[i] = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
        } else {
            *reinterpret_cast<float2*>(p) = make_float2(f[0], f[1]);
        }
    }
}

// E norm weights (plus the offset) from element d on.
template <int E>
__device__ __forceinline__ void load_weights(const void* w, int bf16, float offset, int d, float* out) {
    if (bf16) {
        Chunk<true, E> c;
        c.load(w, d);
        c.widen();
#pragma unroll
        for (int i = 0; i < E; ++i) out[i] = c.f[i] + offset;
    } else {
        Chunk<false, E> c;
        c.load(w, d);
#pragma unroll
        for (int i = 0; i < E; ++i) out[i] = c.f[i] + offset;
    }
}

// The number of i in [1, B] with start[i] <= r: row r's sequence, for a q_start that rises. Wave-uniform.
__device__ __forceinline__ int find_sequence(const int32_t* start, int B, int r) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = B;
    while (n > 0) {
        const int step = (n + 63) / 64;
        const int at = (lane + 1) * step;
        const bool le = at <= n && start[lo + at] <= r;
        const int c = __popcll(__ballot(le));
        lo += c * step;
        n = min(step - 1, n - c * step);
    }
    return lo;
}

template <bool SRC_BF16, bool DST_BF16, int E>
__global__ __launch_bounds__(kThreads) void qkv_append_kernel(QkvAppendArgs a) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6)));
    if (wave == 0 && a.q_start) {  // one wave looks the whole layout over
        for (int i = lane; i <= a.B; i += 64) {
            const int s = a.q_start[i];
            if (s < 0 || s > a.total_q || (i < a.B && a.q_start[i + 1] < s)) latch_error(a.err, ERR_Q_LAYOUT);
        }
    }
    const int r = wave / a.waves_per_row;
    if (r >= a.total_q) return;
    const int head = (wave - r * a.waves_per_row) * (64 >> a.lp_shift) + (lane >> a.lp_shift);
    const int unit = lane & ((1 << a.lp_shift) - 1);
    const int D = a.D;
    // The lane's two chunks (element offsets): unit i < pairs holds i and i + R / 2, the others two
    // neighbouring chunks.
    int d0, d1;
    if (unit < a.pairs) {
        d0 = unit * E;
        d1 = d0 + a.rotary / 2;
    } else {
        d0 = 2 * a.pairs * E + (unit - a.pairs) * 2 * E;
        d1 = d0 + E;
    }
    const bool mine = head < a.H + 2 * a.Hkv;
    const bool has0 = mine && d0 < D, has1 = mine && d1 < D;
    const bool is_q = head < a.H, is_k = !is_q && head < a.H + a.Hkv;
    const int h = is_q ? head : is_k ? head - a.H : head - a.H - a.Hkv;
    const void* src = is_q ? a.query : is_k ? a.key : a.value;
    const size_t from = (size_t)r * (size_t)(is_q ? a.q_stride : is_k ? a.k_stride : a.v_stride) + (size_t)h * D;
    Chunk<SRC_BF16, E> x0, x1;
    x0.zero();
    x1.zero();
    if (has0) x0.load(src, from + d0);
    if (has1) x1.load(src, from + d1);

    // The row's sequence, slot and position.
    int b = r, r0 = r, r1 = r + 1;
    if (a.q_start) {
        b = find_sequence(a.q_start, a.B, r);
        if (b >= a.B) return;  // a row behind the last sequence
        r0 = a.q_start[b];
        r1 = a.q_start[b + 1];
        if (r0 < 0 || r < r0 || r >= r1 || r1 > a.total_q) return;  // before the first, or a bad layout
    }
    const int64_t ctx = a.ctx_lens[b];
    if (ctx < r1 - r0 || ctx > (int64_t)a.max_blocks * a.bs) {
        if (lane == 0) latch_error(a.err, ctx == 0 ? ERR_CTX_EMPTY : ERR_CTX_LEN);
        return;
    }
    const int slot = (int)(ctx - (r1 - r0) + (r - r0));  // below max_blocks * bs, which fits
    const int page = slot / a.bs;
    const int64_t pos = a.positions ? a.positions[r] : slot;
    const int64_t blk = a.table[(size_t)b * a.max_blocks + page];
    const bool bad_pos = a.rotary > 0 && (pos < 0 || pos >= a.max_position);
    const bool bad_blk = blk < 0 || blk >= a.num_blocks;
    if (bad_pos || bad_blk) {
        if (lane == 0) latch_error(a.err, (bad_pos ? ERR_POSITION : 0) | (bad_blk ? ERR_BLOCK_ID : 0));
        return;
    }

    x0.widen();
    x1.widen();
    const bool qk = is_q || is_k;
    if (a.norm) {  // lanes without a chunk hold zeros
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) ss += x0.f[i] * x0.f[i] + x1.f[i] * x1.f[i];
        for (int m = 1; m < (1 << a.lp_shift); m <<= 1) ss += shfl_xor_f(ss, m);
        if (qk) {
            const float rstd = __builtin_amdgcn_rsqf(ss * a.inv_dim + a.eps);
            float w0[E], w1[E];
#pragma unroll
            for (int i = 0; i < E; ++i) w0[i] = w1[i] = 1.f;
            const void* w = is_q ? a.q_weight : a.k_weight;
            if (w) {
                if (has0) load_weights<E>(w, a.weight_bf16, a.weight_offset, d0, w0);
                if (has1) load_weights<E>(w, a.weight_bf16, a.weight_offset, d1, w1);
            }
#pragma unroll
            for (int i = 0; i < E; ++i) {
                x0.f[i] = x0.f[i] * rstd * w0[i];
                x1.f[i] = x1.f[i] * rstd * w1[i];
            }
        }
    }
    if (qk && a.rotary > 0 && mine) {
        const size_t turn = (size_t)pos * (size_t)(a.rotary / 2);
        if (!a.interleaved) {
            if (unit < a.pairs) {
                float c[E], s[E];
                Chunk<false, E>::template load_floats<E>(a.cos + turn + d0, c);
                Chunk<false, E>::template load_floats<E>(a.sin + turn + d0, s);
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const float u = x0.f[i], v = x1.f[i];
                    x0.f[i] = u * c[i] - v * s[i];
                    x1.f[i] = v * c[i] + u * s[i];
                }
            }
        } else {
            float c[E / 2], s[E / 2];
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                float* f = part ? x1.f : x0.f;
                const int d = part ? d1 : d0;
                if (d < a.rotary) {  // rotary is a multiple of E: a chunk turns as a whole or not at all
                    Chunk<false, E>::template load_floats<E / 2>(a.cos + turn + d / 2, c);
                    Chunk<false, E>::template load_floats<E / 2>(a.sin + turn + d / 2, s);
#pragma unroll
                    for (int i = 0; i < E / 2; ++i) {
                        const float u = f[2 * i], v = f[2 * i + 1];
                        f[2 * i] = u * c[i] - v * s[i];
                        f[2 * i + 1] = v * c[i] + u * s[i];
                    }
                }
            }
        }
    }
    if (!mine) return;
    void* dst = is_q ? a.out_query : is_k ? a.kc : a.vc;
    const size_t to = is_q ? ((size_t)r * a.H + h) * D
                           : (((size_t)blk * a.Hkv + h) * a.bs + (size_t)(slot - page * a.bs)) * D;
    if constexpr (SRC_BF16 && DST_BF16) {
        if (!qk) {
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                if (!(part ? has1 : has0)) continue;
                const uint32_t* w = part ? x1.raw : x0.raw;
                uint16_t* p = reinterpret_cast<uint16_t*>(dst) + to + (part ? d1 : d0);
                if constexpr (E == 8) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
                else if constexpr (E == 4) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
                else *reinterpret_cast<uint32_t*>(p) = w[0];
            }
            return;
        }
    }
    if (has0) store_chunk<DST_BF16, E>(dst, to + d0, x0.f);
    if (has1) store_chunk<DST_BF16, E>(dst, to + d1, x1.f);
}

template <int E>
void launch(const QkvAppendArgs& a, unsigned blocks, hipStream_t stream) {
    if (a.src_bf16) {
        if (a.dst_bf16) qkv_append_kernel<true, true, E><<<blocks, kThreads, 0, stream>>>(a);
        else qkv_append_kernel<true, false, E><<<blocks, kThreads, 0, stream>>>(a);
    } else {
        if (a.dst_bf16) qkv_append_kernel<false, true, E><<<blocks, kThreads, 0, stream>>>(a);
        else qkv_append_kernel<false, false, E><<<blocks, kThreads, 0, stream>>>(a);
    }
}

}  // namespace

bool qkv_append_setup(QkvAppendArgs& a) {
    // The widest chunk that the rotation's pairs allow: in halves R / 2 has to be a multiple of it,
    // interleaved R.
    const int unit = a.rotary == 0 ? 8 : a.interleaved ? a.rotary : a.rotary / 2;
    a.chunk = unit % 8 == 0 ? 8 : unit % 4 == 0 ? 4 : 2;
    a.pairs = a.interleaved ? 0 : a.rotary / 2 / a.chunk;
    const int chunks = a.D / a.chunk;
    const int lanes = a.pairs + (chunks - 2 * a.pairs + 1) / 2;
    a.lp_shift = 0;
    while ((1 << a.lp_shift) < lanes) ++a.lp_shift;
    if (a.lp_shift > 6) return false;
    const int heads = 64 >> a.lp_shift;
    const long long all_heads = (long long)a.H + 2ll * a.Hkv;
    if (all_heads > INT32_MAX - 64) return false;  // the kernel counts them in 32 bits
    a.waves_per_row = (int)((all_heads + heads - 1) / heads);
    // A grid has fewer than 2^32 threads.
    constexpr long long kMaxBlocks = (1ll << 32) / kThreads - 1;
    return (long long)a.total_q * a.waves_per_row <= kMaxBlocks * (kThreads / 64);
}

hipError_t launch_qkv_append(const QkvAppendArgs& a, hipStream_t stream) {
    if (a.B == 0 || a.total_q == 0) return hipSuccess;
    const long long waves = (long long)a.total_q * a.waves_per_row;
    const unsigned blocks = (unsigned)((waves + kThreads / 64 - 1) / (kThreads / 64));
    if (a.chunk == 8) launch<8>(a, blocks, stream);
    else if (a.chunk == 4) launch<4>(a, blocks, stream);
    else launch<2>(a, blocks, stream);
    return hipGetLastError();
}

}  // namespace kyro
