// The tiles that the attention kernels for many query rows work on (prefill_attention.hip, shared_attention.hip): K and
// V of 64 or 32 tokens of one kv head in LDS, a wave's 32 query rows in registers, and the products between them in
// the 32 x 32 MFMA layout. S^T = K Q^T puts a query row in one lane pair (l, l + 32), and its fragment is already the
// P^T operand of O^T += V^T P^T. (prefill_attention.hip has the products in its own loop: as functions they cost its
// instances at wide heads other registers than they are tuned for.)
#pragma once

#include "attention_rows.hpp"

namespace kyro {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kPfThreads = 256;
constexpr int kPfWaves = kPfThreads / 64;
constexpr int kPfBS = 16;  // tokens per slot (slab) of the cache
constexpr int kRawWord3 = 0x00020000;

// Read in place of a missing slab; never written.
__device__ uint4 kPfZeroSlab[kPfBS * 512 / 16];

// Layout of a head dim DR (a multiple of 16) with 2- or 4-byte elements.
template <bool BF16, int DR>
struct PfCfg {
    static constexpr bool BF = BF16;
    static constexpr int R = DR;
    static constexpr int ES = BF16 ? 2 : 4;
    static constexpr int D = (DR + 31) / 32 * 32;    // columns of V and O held (padded to 32)
    static constexpr int DT = D / 32;                // 32-column tiles of O^T
    static constexpr int KS = DR * ES / 32;          // 32-byte steps of a K or Q row
    static constexpr int CPR = DR * ES / 16;         // 16-byte chunks of a cache row
    static constexpr int NCH = D * ES / 16;          // chunk slots of a row in LDS
    // LDS slab: [NCH / CW column groups][16 tokens][CW chunks]. One copy instruction fills 64
    // consecutive chunks: 4 whole 256-byte rows at CW = 16.
    static constexpr int CW = NCH % 16 == 0 ? 16 : NCH % 8 == 0 ? 8 : 4;
    static constexpr int SLAB = kPfBS * NCH;         // chunks of a slab
    static constexpr int TK = prefill_tile_tokens(BF16, DR);
    static constexpr int NS = TK / kPfBS;            // slabs of a tile
    static constexpr int TT = TK / 32;               // 32-token tiles of S^T
    // f32 head dims where the kernel stands in for the vector kernel, whose sums are trees: short chains
    // of additions (8 in a score, 4 in a tile's O^T += V^T P^T) that are added up in two halves. The error
    // against 64 bits is then level with the vector kernel's over 33 to 4000 tokens (prompts of 200 tokens,
    // head dims 64 / 80 / 96 / 112, 1e-7: 1.15 1.22 1.24 1.23 here, 1.16 1.22 1.26 1.23 there; with two
    // chains per score, as at 128, 1.82 at 112). At head dim 128 two long chains per score and one per
    // output are already closer than the one-block kernel's single chain (1.89 against 2.80). Over shared prefixes (160
    // sequences of 400 tokens, the same head dims; chains of 8 in a score, 4 in an output): 1.75 1.87 1.89 1.85 here, 1.76
    // 1.84 1.92 1.87 there; 2.23 2.49 2.56 2.62 with the chains of head dim 128, which are 1.03 to 1.11 times as fast.
    static constexpr bool TREE = !BF16 && DR < 128;
    // K rows: chunk c of token t sits in slot c ^ swk(t) of its column group, so that the 16
    // tokens of an operand read (same c) spread over all banks.
    __device__ static constexpr int swk(int t) { return t * CW / 16; }
    // V rows (bf16): the transposing loads of lanes 0..31 take 64 bytes of each of 4 consecutive
    // tokens; slot c ^ swv(t) puts those on distinct banks. f32 V is read 128 bytes of one token
    // at a time: no swizzle.
    __device__ static constexpr int swv(int t) { return BF16 ? 4 * ((t * CW / 16) & (CW / 4 - 1)) : 0; }
    static_assert(DR % 16 == 0 && NCH % 4 == 0, "rows of whole 16-byte chunks");
    static_assert((NS == 4 || NS == 2) && kPfBS * DR * ES <= (int)sizeof(kPfZeroSlab), "tile shape");
};

// One of the C::SLAB / 64 copies of 64 consecutive chunks that take a slab (16 tokens of one kv head, `from`) into LDS
// at dst (wave-uniform). V selects the V swizzle. Columns past the head dim (DR < D) repeat the row's last chunk: K's are
// never read, V's reach only output columns that are not stored.
template <class C, bool V, int POL>
__device__ __forceinline__ void copy_chunks(uint4* dst, __amdgpu_buffer_rsrc_t from, int lane, int e) {
    constexpr int kGroup = kPfBS * C::CW;  // chunks of a column group (a multiple of 64)
    const int cg = 64 * e / kGroup;
    const int pos = 64 * e - cg * kGroup + lane;
    const int t = pos / C::CW;
    const int slot = pos % C::CW;
    int c = cg * C::CW + (slot ^ (V ? C::swv(t) : C::swk(t)));
    if (C::CPR < C::NCH) c = min(c, C::CPR - 1);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)(dst + 64 * e), 16,
                                             (t * C::CPR + c) * 16, 0, 0, POL);
}

// A slab as a buffer; one of no bytes reads as zeros.
template <class C>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t slab_buffer(const void* base, bool empty = false) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, empty ? 0 : kPfBS * C::CPR * 16, kRawWord3);
}

template <class C, bool V, int POL>
__device__ __forceinline__ void copy_slab(uint4* dst, const void* base, int lane) {
    const __amdgpu_buffer_rsrc_t r = slab_buffer<C>(base);
#pragma unroll
    for (int e = 0; e < C::SLAB / 64; ++e) copy_chunks<C, V, POL>(dst, r, lane, e);
}

// Operand addresses (bytes) of a lane in a tile, one per swizzle pattern.
template <class C>
struct TileLane {
    int k[C::CW / 2];
    int v[C::CW / 4];
    int v32;
    __device__ explicit TileLane(int lane) {
        const int h = lane >> 5, i16 = lane & 15;
#pragma unroll
        for (int x = 0; x < C::CW / 2; ++x)
            k[x] = ((lane >> 4) & 1) * (C::SLAB * 16) + (lane & 15) * (C::CW * 16) + ((2 * x + h) ^ C::swk(lane & 15)) * 16;
        const int tok = C::BF ? 4 * h + (i16 >> 2) : 4 * h;
#pragma unroll
        for (int x = 0; x < C::CW / 4; ++x)
            v[x] = C::BF ? tok * (C::CW * 16) + ((2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1)) ^ C::swv(tok) ^ (4 * x)) * 16 + 8 * (i16 & 1) : 0;
        v32 = tok * (C::CW * 16) + 4 * (lane & 31);
    }
};

template <class C>
constexpr int kTileGroupBytes = kPfBS * C::CW * 16;  // a column group of a slab

// 32-byte step s of K's operand for the 32 tokens of tt of a tile at kb in LDS.
template <class C>
__device__ __forceinline__ uint4 k_operand(const char* kb, const TileLane<C>& at, int tt, int s) {
    return *reinterpret_cast<const uint4*>(kb + at.k[s % (C::CW / 2)] + 2 * tt * (C::SLAB * 16) + (2 * s / C::CW) * kTileGroupBytes<C>);
}

// bf16 V^T of 16 tokens (y of the 32 of tt) and columns 32 dt .. of a tile at vb.
template <class C>
__device__ __forceinline__ uint4 v_operand(const char* vb, const TileLane<C>& at, int tt, int y, int dt) {
    const char* va = vb + at.v[dt % (C::CW / 4)] + (2 * tt + y) * (C::SLAB * 16) + (4 * dt / C::CW) * kTileGroupBytes<C>;
    using Ptr = __attribute__((address_space(3))) s16x4*;
    const uint2 lo = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(va)));
    const uint2 hi = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(va + 8 * C::CW * 16)));
    return make_uint4(lo.x, lo.y, hi.x, hi.y);
}

__device__ __forceinline__ f32x16 mfma_bf16(const uint4& x, const uint4& y, const f32x16& z) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), z, 0, 0, 0);
}

__device__ __forceinline__ f32x16 zeros() {
    f32x16 z;
#pragma unroll
    for (int x = 0; x < 16; ++x) z[x] = 0.f;
    return z;
}

// S^T of 32 tokens (those of tt) of a tile: K at kb in LDS, the wave's rows in q.
template <class C>
__device__ __forceinline__ f32x16 tile_scores(const char* kb, const uint4* q, const TileLane<C>& at, int tt) {
    if constexpr (C::BF) {
        f32x16 sum = zeros();
#pragma unroll
        for (int s = 0; s < C::KS; ++s)
            sum = mfma_bf16(k_operand<C>(kb, at, tt, s), q[s], sum);
        // Keep operand reads in flight ahead of the products (the compiler's own order waits for each).
        constexpr int kAhead = C::R < 256 ? 4 : 1;
        __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
        for (int x = 0; x < C::KS - kAhead; ++x) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, kAhead, 0);
        return sum;
    } else {
        // Two chains of additions; with TREE two new ones of eight for every four steps, which are then added up.
        constexpr int kSteps = C::TREE ? 4 : C::KS;
        f32x16 sum, chain[2] = {zeros(), zeros()};
#pragma unroll
        for (int s = 0; s < C::KS; ++s) {
            const f32x4 kf = __builtin_bit_cast(f32x4, k_operand<C>(kb, at, tt, s));
            f32x4 qf = __builtin_bit_cast(f32x4, q[s]);
            if (s > 0 && s % kSteps == 0) {
                // The products behind depend on the sum before them. Left alone the compiler puts all additions at the
                // end, with every chain in registers of its own: 295 spilled at head dim 112, where this spills none.
                float q0 = qf[0], q1 = qf[1];
                asm volatile("" : "+v"(sum), "+v"(q0), "+v"(q1));
                qf[0] = q0;
                qf[1] = q1;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) chain[e % 2] = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[e], qf[e], chain[e % 2], 0, 0, 0);
            if ((s + 1) % kSteps != 0 && s + 1 < C::KS) continue;
            if (s < kSteps) sum = chain[0] + chain[1];
            else sum += chain[0] + chain[1];
            chain[0] = chain[1] = zeros();
        }
        return sum;
    }
}

// 32 tokens' weights as the bf16 operands of their products, 16 tokens each.
__device__ __forceinline__ void tile_weights(const f32x16& p, uint4* w) {
#pragma unroll
    for (int y = 0; y < 2; ++y)
        w[y] = make_uint4(pack_bf16x2(p[8 * y], p[8 * y + 1]), pack_bf16x2(p[8 * y + 2], p[8 * y + 3]),
                          pack_bf16x2(p[8 * y + 4], p[8 * y + 5]), pack_bf16x2(p[8 * y + 6], p[8 * y + 7]));
}

// O^T += V^T P^T over 32 tokens (those of tt) of a tile: V at vb in LDS, the weights in w4 (bf16) or p.
template <class C>
__device__ __forceinline__ void tile_output(const char* vb, const f32x16& p, const uint4* w4, const TileLane<C>& at, f32x16* o, int tt) {
    if constexpr (C::BF) {
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int dt = 0; dt < C::DT; ++dt) o[dt] = mfma_bf16(v_operand<C>(vb, at, tt, y, dt), w4[y], o[dt]);
    } else {
        // A tile's products are summed on their own and then added: the chain of additions into O^T is one per tile
        // instead of one per two tokens.
        // With TREE that sum is one of four chains of four, two at a time.
        auto product = [&](int dt, int x, const f32x16& to) -> f32x16 {
            const float vv = *reinterpret_cast<const float*>(vb + at.v32 + (2 * tt + x / 8) * (C::SLAB * 16) + (8 * dt / C::CW) * kTileGroupBytes<C> +
                                                             (8 * ((x / 4) % 2) + x % 4) * (C::CW * 16) + (8 * dt % C::CW) * 16);
            return __builtin_amdgcn_mfma_f32_32x32x2f32(vv, p[x], to, 0, 0, 0);
        };
        if constexpr (C::TREE) {
#pragma unroll
            for (int dt = 0; dt < C::DT; ++dt) {
                f32x16 sum;
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    f32x16 chain[2] = {zeros(), zeros()};
#pragma unroll
                    for (int x = 8 * y; x < 8 * y + 8; ++x) chain[x % 2] = product(dt, x, chain[x % 2]);
                    if (y == 0) sum = chain[0] + chain[1];
                    else sum += chain[0] + chain[1];
                    __builtin_amdgcn_sched_barrier(0);
                }
                o[dt] += sum;
            }
        } else {
            constexpr int W = 2;  // column tiles side by side
#pragma unroll
            for (int d0 = 0; d0 < C::DT; d0 += W) {
                f32x16 sum[W];
#pragma unroll
                for (int w = 0; w < W; ++w) sum[w] = zeros();
#pragma unroll
                for (int x = 0; x < 16; ++x)
#pragma unroll
                    for (int w = 0; w < W; ++w)
                        if (d0 + w < C::DT) sum[w] = product(d0 + w, x, sum[w]);
#pragma unroll
                for (int w = 0; w < W; ++w)
                    if (d0 + w < C::DT) o[d0 + w] += sum[w];
            }
        }
    }
}

}  // namespace

}  // namespace kyro
