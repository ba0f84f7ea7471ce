// decode_int4.cuh — single-token decode attention over a 4-bit KV cache
// (format: kv_int4.cuh) for sm_100a, with grouped query heads and a length
// for every sequence.
//
//   O[b,h,:] = sum_t softmax_t(q_bh . k_t / sqrt(D)) v_t,   t < length[b]
//   k_t[i] = code * scale + zero of element i's block, v_t likewise
//
// Bound: HBM.  A row pair is D codes bytes plus 8 D / BS bytes of parameters, so
// at 6.5 TB/s an SM must take in ~46 codes a clock.  Unpacking each code to a
// float for CUDA-core FMAs would cost more issue slots than there are, for
// every query head again; so the products run on the tensor cores with the
// codes as they are.  The matrix shapes are (16 tokens x 16 elements) x (16 x
// 8 query heads) and the products take the same time for 1 to 8 heads; tcgen05
// would have to write the expanded codes to shared memory or TMEM first, for
// an M of which one head uses 1 / 128, so the products are warp-level mma.
//
// Codes as fp16 without conversion.  A nibble in the low bits of a 16-bit
// half IS the fp16 subnormal code * 2^-24, and one in bits 4..7 is code *
// 2^-20: one AND yields two operands, products with them are exact, sums are
// fp32.  q is scaled by a power of two per head (exact) and by 2^-4 where it
// meets the second kind.
//   score_t = sum_blocks scale_t (codes . q) + zero_t (sum of q over the block)
//   O       = [ sum_t (p_t scale_t) codes_t + sum_t p_t zero_t ] / sum_t p_t
// The block scale is applied to the score in fp32; for V it is multiplied into
// p in fp32 before p is rounded to fp16 as the product's operand (relative
// error 2^-12 a token, like the 16-bit P of any tensor-core attention).  The
// zero sums stay in fp32.
//
// Range.  p * scale must stay inside fp16 whatever the caches hold, so the
// running reference of the softmax is M >= max_t(score_t + log2 of the scale's
// upper power of two), in base 2, and the operand is 2^(score - M + 11) *
// scale < 2^11; M moves only when a token exceeds it by 2^4.
//
// Work split.  Units are (sequence, KV head, slice of 8 * NT query heads); a
// unit has ceil(length / TILE) tiles.  All units' tiles, end to end, are cut
// into equal runs, one per CTA, whatever the lengths are; the CTA's 4 warps
// take its tiles in turn.  A unit that lies in one CTA is finished there; of a
// unit cut across CTAs each leaves a record (acc[D], M, l per query head) in
// the workspace, and the CTA that arrives last at the unit's counter merges
// the records in order: the result does not depend on which one that is.
// Records and counters are zeroed again by the CTA that merges.
//
// Every warp streams for itself: a ring of STAGES tiles, K and V rows by bulk
// copies (one lane), the parameters by one cp.async per row, which fills rows
// behind the sequence's end with zeros: their codes are whatever the buffer
// held (any 4 bits are finite), their weights are zero, and rows past the
// length are never read.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "device_common.cuh"
#include "kv_int4.cuh"

namespace tqkv {

constexpr int kI4Warps = 4;
constexpr int kI4Threads = kI4Warps * 32;

struct Int4DecodeArgs {
    const uint16_t* q;          // [B, Hq, D]
    const uint8_t *kq, *vq;     // [B, Hkv, S_cap, D / 2]
    const uint32_t *ks, *vs;    // [B, Hkv, S_cap, D / BS] (scale, zero)
    uint16_t* o;                // [B, Hq, D]
    const int32_t* lengths;     // [B], or null: S for every sequence
    unsigned int* counters;     // one per CTA
    float* recs;                // [CTA][2][rows][D + 4]
    long long S_cap;
    int B, Hq, Hkv, group, slices, S;
    int rec_rows;               // query heads a record holds: min(group, 8 * NT)
    int min_tiles;              // tiles a CTA takes at least
    int stream_once;            // L2: the cache will not be read again soon
    float score_scale;          // log2(e) / sqrt(D)
};

template <int D, int BS, int NT>
struct I4Cfg {
    static constexpr int kRow = D / 2;            // bytes of codes a row
    static constexpr int kSub = D / 32;           // 32-element groups = words per lane chunk
    static constexpr int kNS = D / BS;            // blocks a row
    static constexpr int kTile = 4096 / D;        // rows a tile: 2 KB of codes
    static constexpr int kM = kTile / 16;         // 16-row pieces
    static constexpr int kQ = 8 * NT;             // query heads a unit takes
    static constexpr int kKV = kTile * kRow;
    static constexpr int kSc = kTile * kNS * 4;
    static constexpr int kStage = 2 * (kKV + kSc);
    static constexpr int kStages = 3;
    static constexpr int kRing = kI4Warps * kStages * kStage;
    static constexpr int kRecStride = D + 4;      // acc[D], l at D, M at D + 1
    static constexpr int kOffMerge = kRing + kI4Warps * kStages * 8 + 16;
    static_assert(kOffMerge % 16 == 0, "alignment");
    static int smem_bytes(int rows) { return kOffMerge + kI4Warps * rows * kRecStride * 4; }
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// transpose of an 8 x 8 matrix of 16-bit values held two to a lane
__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}

// `bytes` (4, 8 or 16) of global memory into shared memory, or zeros
template <int bytes>
__device__ __forceinline__ void cp_async_zfill(uint32_t dst, const void* src, bool real) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(bytes),
                 "r"(real ? bytes : 0)
                 : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(bar))
                 : "memory");
}

// bulk copy without an L2 hint
__device__ __forceinline__ void bulk_copy_g2s_plain(void* dst, const void* src, uint32_t bytes,
                                                    uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
            smem_addr(dst)),
        "l"(src), "r"(bytes), "r"(smem_addr(bar))
        : "memory");
}

__device__ __forceinline__ int i4_length(const Int4DecodeArgs& a, int b) {
    if (a.lengths == nullptr) return a.S;
    const int n = a.lengths[b];
    return n < 0 ? 0 : n > a.S ? a.S : n;
}

// The unit that a tile belongs to, moved forward tile by tile.
template <int TILE>
struct UnitWalk {
    int b, u;         // sequence; (KV head, slice) within it
    int len, nt;      // its rows and tiles
    long long start;  // first tile of the unit

    __device__ __forceinline__ void load(const Int4DecodeArgs& a) {
        len = b < a.B ? i4_length(a, b) : 0;
        nt = (len + TILE - 1) / TILE;
    }
    // g below the total: the loop ends
    __device__ __forceinline__ void seek(const Int4DecodeArgs& a, long long g) {
        while (g >= start + nt && b < a.B) {
            start += nt;
            if (nt > 0 && ++u < a.Hkv * a.slices) continue;
            u = 0;
            ++b;
            load(a);
        }
    }
};

template <int D, int BS, int NT>
__global__ void __launch_bounds__(kI4Threads, NT == 1 ? 4 : 2)
    decode_int4_kernel(Int4DecodeArgs a, int bf16) {
    using C = I4Cfg<D, BS, NT>;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, c = lane & 3;  // the mma's row and column groups
    uint8_t* ring = smem + warp * C::kStages * C::kStage;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kRing) + warp * C::kStages;
    unsigned int* flag = reinterpret_cast<unsigned int*>(smem + C::kRing + kI4Warps * C::kStages * 8);
    float* merge = reinterpret_cast<float*>(smem + C::kOffMerge);

    if (lane == 0) {
        for (int i = 0; i < C::kStages; ++i) mbar_init(bars + i, 33);  // 32 lanes' parameters, 1 codes
        fence_barrier_init();
    }
    __syncwarp();
    griddep_wait();
    griddep_launch_dependents();

    // ---- this CTA's tiles [g0, g1) of all units' n
    const int per_seq = a.Hkv * a.slices;
    long long n = 0;
    if (a.lengths == nullptr) {
        n = static_cast<long long>(a.B) * per_seq * ((a.S + C::kTile - 1) / C::kTile);
    } else {
        for (int b = lane; b < a.B; b += 32) n += (i4_length(a, b) + C::kTile - 1) / C::kTile;
#pragma unroll
        for (int off = 16; off; off >>= 1) n += __shfl_xor_sync(0xffffffffu, n, off);
        n *= per_seq;
    }
    // heads of sequences that hold nothing come out as zero
    if (a.lengths != nullptr || a.S == 0) {
        for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
            if (i4_length(a, b) != 0) continue;
            uint32_t* o = reinterpret_cast<uint32_t*>(a.o) + static_cast<long long>(b) * a.Hq * (D / 2);
            for (int i = threadIdx.x; i < a.Hq * (D / 2); i += kI4Threads) o[i] = 0u;
        }
    }
    long long ctas = n / a.min_tiles;
    if (ctas > gridDim.x) ctas = gridDim.x;
    if (ctas < 1) ctas = 1;
    const long long cta = blockIdx.x;
    if (cta >= ctas || n == 0) return;
    const long long g0 = n * cta / ctas, g1 = n * (cta + 1) / ctas;
    auto cta_of = [&](long long tile) { return ((tile + 1) * ctas - 1) / n; };

    UnitWalk<C::kTile> walk;  // of the unit being worked on
    if (a.lengths == nullptr) {
        const int nt = (a.S + C::kTile - 1) / C::kTile;
        const long long unit = g0 / nt;
        walk.b = static_cast<int>(unit / per_seq);
        walk.u = static_cast<int>(unit - static_cast<long long>(walk.b) * per_seq);
        walk.start = unit * nt;
        walk.load(a);
    } else {
        walk.start = 0;
        walk.b = 0;
        for (int base = 0; base < a.B; base += 32) {
            const int b = base + lane;
            long long x = b < a.B ? static_cast<long long>((i4_length(a, b) + C::kTile - 1) / C::kTile) * per_seq
                                  : 0;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const long long y = __shfl_up_sync(0xffffffffu, x, off);
                if (lane >= off) x += y;
            }
            const unsigned past = __ballot_sync(0xffffffffu, walk.start + x <= g0);
            const int k = __popc(past);  // sequences of these 32 that end at or before g0
            if (k > 0) {
                walk.start += __shfl_sync(0xffffffffu, x, k - 1);
                walk.b = base + k;
            }
            if (k < 32) break;
        }
        walk.load(a);
        const long long in = g0 - walk.start;
        walk.u = static_cast<int>(in / walk.nt);
        walk.start += static_cast<long long>(walk.u) * walk.nt;
    }

    // ---- this warp's stream of tiles: g0 + warp, g0 + warp + 4, ...
    const uint64_t policy = make_evict_first_policy();
    UnitWalk<C::kTile> ahead = walk;
    long long next = g0 + warp;
    int issued = 0;
    auto issue = [&]() {
        if (next >= g1) return;
        ahead.seek(a, next);
        const int st = issued % C::kStages;
        uint8_t* buf = ring + st * C::kStage;
        uint64_t* bar = bars + st;
        const int t0 = static_cast<int>(next - ahead.start) * C::kTile;
        const int rows = ahead.len - t0 < C::kTile ? ahead.len - t0 : C::kTile;
        const int h = ahead.u / a.slices;
        const long long row = (static_cast<long long>(ahead.b) * a.Hkv + h) * a.S_cap + t0;
        if (lane == 0) {
            const uint32_t bytes = rows * C::kRow;
            mbar_arrive_expect_tx(bar, 2 * bytes);
            if (a.stream_once) {
                bulk_copy_g2s(buf, a.kq + row * C::kRow, bytes, bar, policy);
                bulk_copy_g2s(buf + C::kKV, a.vq + row * C::kRow, bytes, bar, policy);
            } else {
                bulk_copy_g2s_plain(buf, a.kq + row * C::kRow, bytes, bar);
                bulk_copy_g2s_plain(buf + C::kKV, a.vq + row * C::kRow, bytes, bar);
            }
        }
        const uint32_t sc = smem_addr(buf + 2 * C::kKV);
#pragma unroll
        for (int r = lane; r < C::kTile; r += 32) {
            const bool real = r < rows;
            const long long p = (row + (real ? r : 0)) * C::kNS;
            cp_async_zfill<4 * C::kNS>(sc + r * 4 * C::kNS, a.ks + p, real);
            cp_async_zfill<4 * C::kNS>(sc + C::kSc + r * 4 * C::kNS, a.vs + p, real);
        }
        cp_async_arrive(bar);
        ++issued;
        next += kI4Warps;
    };
    for (int i = 0; i < C::kStages; ++i) issue();

    int taken = 0;
    bool dead = false;  // a wait ran out: the results become NaN, nothing more is waited for
    long long mine = g0 + warp;

    for (long long p0 = g0; p0 < g1;) {
        // ---- one piece: the CTA's tiles [p0, p1) of one unit
        walk.seek(a, p0);
        const long long unit_end = walk.start + walk.nt;
        const long long p1 = unit_end < g1 ? unit_end : g1;
        const int kvh = walk.u / a.slices, slice = walk.u - kvh * a.slices;
        const int head0 = kvh * a.group + slice * C::kQ;
        const int nq = a.group - slice * C::kQ < C::kQ ? a.group - slice * C::kQ : C::kQ;

        // ---- q of the unit as the products' right operands
        uint32_t qf[NT][C::kSub][2][2];
        float qsum[NT][C::kNS][2], sc[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const bool has = t * 8 + g < nq;
            float f[C::kSub][8];
            float amax = 0.0f;
            const uint4* src = reinterpret_cast<const uint4*>(
                a.q + (static_cast<long long>(walk.b) * a.Hq + head0 + (has ? t * 8 + g : 0)) * D);
#pragma unroll
            for (int b = 0; b < C::kSub; ++b) {
                uint4 raw = make_uint4(0, 0, 0, 0);
                if (has) raw = src[b * 4 + c];
                if (bf16) unpack8<true>(raw, f[b]);
                else unpack8<false>(raw, f[b]);
#pragma unroll
                for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(f[b][i]));
            }
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            // 2^e with max |q| * 2^e in [2^10, 2^11): exact in fp16 down to
            // 2^-24 of the largest element
            int e = 137 - static_cast<int>(__float_as_uint(amax) >> 23);
            e = amax == 0.0f || amax > 3.0e38f ? 0 : e > 100 ? 100 : e < -100 ? -100 : e;
            const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
            float sum[C::kNS];
#pragma unroll
            for (int s = 0; s < C::kNS; ++s) sum[s] = 0.0f;
#pragma unroll
            for (int b = 0; b < C::kSub; ++b) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    f[b][i] *= up;
                    sum[b * 32 / BS] += f[b][i];
                }
                // elements 0, 4, 2, 6 meet codes * 2^-24, elements 1, 5, 3, 7 codes * 2^-20
                qf[t][b][0][0] = pack2<false>(f[b][0], f[b][4]);
                qf[t][b][0][1] = pack2<false>(f[b][2], f[b][6]);
                qf[t][b][1][0] = pack2<false>(f[b][1] * 0.0625f, f[b][5] * 0.0625f);
                qf[t][b][1][1] = pack2<false>(f[b][3] * 0.0625f, f[b][7] * 0.0625f);
            }
            // the scores' columns in this lane are heads 2c and 2c + 1
#pragma unroll
            for (int s = 0; s < C::kNS; ++s) {
                sum[s] += __shfl_xor_sync(0xffffffffu, sum[s], 1);
                sum[s] += __shfl_xor_sync(0xffffffffu, sum[s], 2);
                sum[s] *= 5.9604644775390625e-08f;  // 2^-24, as the codes
                qsum[t][s][0] = __shfl_sync(0xffffffffu, sum[s], 8 * c);
                qsum[t][s][1] = __shfl_sync(0xffffffffu, sum[s], 8 * c + 4);
            }
            const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23) * 16777216.0f *
                               a.score_scale;
            sc[t][0] = __shfl_sync(0xffffffffu, down, 8 * c);
            sc[t][1] = __shfl_sync(0xffffffffu, down, 8 * c + 4);
        }

        float acc[NT][C::kSub][2][4], zsum[NT][C::kNS][2], M[NT][2], l[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int b = 0; b < C::kSub; ++b)
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[t][b][i >> 2][i & 3] = 0.0f;
#pragma unroll
            for (int s = 0; s < C::kNS; ++s) zsum[t][s][0] = zsum[t][s][1] = 0.0f;
            M[t][0] = M[t][1] = -INFINITY;
            l[t][0] = l[t][1] = 0.0f;
        }

        // ---- the warp's tiles of the piece
        for (; mine < p1; mine += kI4Warps) {
            const int st = taken % C::kStages;
            const uint8_t* buf = ring + st * C::kStage;
            if (!dead && !mbar_wait_bounded(bars + st, (taken / C::kStages) & 1)) {
                dead = true;
                if (lane == 0) record_device_error(kErrFullWaitTimeout);
            }
            dead = __any_sync(0xffffffffu, dead);
            const int left = walk.len - static_cast<int>(mine - walk.start) * C::kTile;
            const uint32_t* kp = reinterpret_cast<const uint32_t*>(buf + 2 * C::kKV);
            const uint32_t* vp = kp + C::kSc / 4;

            // scores of the tile, in units where 2^(x * sc) is the weight
            float s[NT][C::kM][4];
#pragma unroll
            for (int m = 0; m < C::kM; ++m) {
                uint32_t w0[C::kSub], w1[C::kSub];
                const uint8_t* r0 = buf + (m * 16 + g) * C::kRow + c * (C::kRow / 4);
                if constexpr (C::kSub == 4) {
                    *reinterpret_cast<uint4*>(w0) = *reinterpret_cast<const uint4*>(r0);
                    *reinterpret_cast<uint4*>(w1) = *reinterpret_cast<const uint4*>(r0 + 8 * C::kRow);
                } else {
                    *reinterpret_cast<uint2*>(w0) = *reinterpret_cast<const uint2*>(r0);
                    *reinterpret_cast<uint2*>(w1) = *reinterpret_cast<const uint2*>(r0 + 8 * C::kRow);
                }
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[t][m][i] = 0.0f;
                float d[NT][4];
#pragma unroll
                for (int b = 0; b < C::kSub; ++b) {
                    if (b % (BS / 32) == 0) {
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int i = 0; i < 4; ++i) d[t][i] = 0.0f;
                    }
                    const uint32_t v0 = w0[b] >> 8, v1 = w1[b] >> 8;
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        mma_f16(d[t], w0[b] & 0x000f000fu, w1[b] & 0x000f000fu, v0 & 0x000f000fu,
                                v1 & 0x000f000fu, qf[t][b][0][0], qf[t][b][0][1]);
                        mma_f16(d[t], w0[b] & 0x00f000f0u, w1[b] & 0x00f000f0u, v0 & 0x00f000f0u,
                                v1 & 0x00f000f0u, qf[t][b][1][0], qf[t][b][1][1]);
                    }
                    if ((b + 1) % (BS / 32) == 0) {
                        const int blk = b * 32 / BS;
                        const uint32_t p0w = kp[(m * 16 + g) * C::kNS + blk];
                        const uint32_t p1w = kp[(m * 16 + g + 8) * C::kNS + blk];
                        const float2 a0 = __half22float2(*reinterpret_cast<const __half2*>(&p0w));
                        const float2 a1 = __half22float2(*reinterpret_cast<const __half2*>(&p1w));
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            s[t][m][0] = fmaf(d[t][0], a0.x, fmaf(a0.y, qsum[t][blk][0], s[t][m][0]));
                            s[t][m][1] = fmaf(d[t][1], a0.x, fmaf(a0.y, qsum[t][blk][1], s[t][m][1]));
                            s[t][m][2] = fmaf(d[t][2], a1.x, fmaf(a1.y, qsum[t][blk][0], s[t][m][2]));
                            s[t][m][3] = fmaf(d[t][3], a1.x, fmaf(a1.y, qsum[t][blk][1], s[t][m][3]));
                        }
                    }
                }
            }
            if (left < C::kTile) {
#pragma unroll
                for (int m = 0; m < C::kM; ++m)
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        if (m * 16 + g >= left) s[t][m][0] = s[t][m][1] = -INFINITY;
                        if (m * 16 + g + 8 >= left) s[t][m][2] = s[t][m][3] = -INFINITY;
                    }
            }

            // ---- reference of the weights
            float vsc[C::kM][2][C::kNS], vz[C::kM][2][C::kNS];
            float top[NT][2];
#pragma unroll
            for (int t = 0; t < NT; ++t) top[t][0] = top[t][1] = -INFINITY;
#pragma unroll
            for (int m = 0; m < C::kM; ++m)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float big = 0.0f;
#pragma unroll
                    for (int k = 0; k < C::kNS; ++k) {
                        const uint32_t pw = vp[(m * 16 + g + 8 * r) * C::kNS + k];
                        const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&pw));
                        vsc[m][r][k] = p.x;
                        vz[m][r][k] = p.y;
                        big = fmaxf(big, p.x);
                    }
                    // exponent of the power of two above the scale, at least
                    // -24 (fp16's smallest step; blocks of one value have scale 0)
                    const float et = fmaxf(
                        __uint_as_float(0x4b000000u | (__float_as_uint(big) >> 23)) - 8388734.0f,
                        -24.0f);
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int j = 0; j < 2; ++j)
                            top[t][j] = fmaxf(top[t][j], fmaf(s[t][m][2 * r + j], sc[t][j], et));
                }
            bool over = false;
#pragma unroll
            for (int t = 0; t < NT; ++t) over |= top[t][0] > M[t][0] + 4.0f || top[t][1] > M[t][1] + 4.0f;
            if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float x = top[t][j];
#pragma unroll
                        for (int off = 4; off < 32; off <<= 1)
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
                        x = fmaxf(x, M[t][j]);
                        const float f = x == M[t][j] ? 1.0f : fast_exp2(M[t][j] - x);
                        M[t][j] = x;
                        l[t][j] *= f;
#pragma unroll
                        for (int k = 0; k < C::kNS; ++k) zsum[t][k][j] *= f;
#pragma unroll
                        for (int b = 0; b < C::kSub; ++b) {
                            acc[t][b][0][j] *= f;
                            acc[t][b][0][j + 2] *= f;
                            acc[t][b][1][j] *= f;
                            acc[t][b][1][j + 2] *= f;
                        }
                    }
            }

            // ---- weights and the second product
#pragma unroll
            for (int m = 0; m < C::kM; ++m) {
                uint32_t bw[NT][C::kNS][2];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    float p[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        p[i] = fast_exp2(fmaf(s[t][m][i], sc[t][i & 1], 11.0f - M[t][i & 1]));
                    l[t][0] += p[0] + p[2];
                    l[t][1] += p[1] + p[3];
#pragma unroll
                    for (int k = 0; k < C::kNS; ++k) {
                        bw[t][k][0] = movmatrix(pack2<false>(p[0] * vsc[m][0][k], p[1] * vsc[m][0][k]));
                        bw[t][k][1] = movmatrix(pack2<false>(p[2] * vsc[m][1][k], p[3] * vsc[m][1][k]));
                        zsum[t][k][0] = fmaf(p[0], vz[m][0][k], fmaf(p[2], vz[m][1][k], zsum[t][k][0]));
                        zsum[t][k][1] = fmaf(p[1], vz[m][0][k], fmaf(p[3], vz[m][1][k], zsum[t][k][1]));
                    }
                }
                // tokens 2c, 2c + 1, 2c + 8, 2c + 9 of the piece; this lane's 16
                // bits of each 32-element group
                const uint8_t* v0 = buf + C::kKV + (m * 16 + 2 * c) * C::kRow + (g >> 1) * (C::kRow / 4);
                uint32_t x[4][C::kSub];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint8_t* src = v0 + ((i & 1) + (i >> 1) * 8) * C::kRow;
                    if constexpr (C::kSub == 4)
                        *reinterpret_cast<uint4*>(x[i]) = *reinterpret_cast<const uint4*>(src);
                    else
                        *reinterpret_cast<uint2*>(x[i]) = *reinterpret_cast<const uint2*>(src);
                }
                const uint32_t sel = (g & 1) ? 0x7632u : 0x5410u;
#pragma unroll
                for (int b = 0; b < C::kSub; ++b) {
                    const int k = b * 32 / BS;
                    const uint32_t lo = __byte_perm(x[0][b], x[1][b], sel);
                    const uint32_t hi = __byte_perm(x[2][b], x[3][b], sel);
                    const uint32_t lo8 = lo >> 8, hi8 = hi >> 8;
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        mma_f16(acc[t][b][0], lo & 0x000f000fu, lo8 & 0x000f000fu, hi & 0x000f000fu,
                                hi8 & 0x000f000fu, bw[t][k][0], bw[t][k][1]);
                        mma_f16(acc[t][b][1], lo & 0x00f000f0u, lo8 & 0x00f000f0u, hi & 0x00f000f0u,
                                hi8 & 0x00f000f0u, bw[t][k][0], bw[t][k][1]);
                    }
                }
            }
            ++taken;
            __syncwarp();  // every lane is done with the stage: refill it
            if (!dead) issue();
        }

        // ---- the warp's state to shared memory: acc[D], l, M per query head
        const int rows = a.rec_rows;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float ls = l[t][j];
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) ls += __shfl_xor_sync(0xffffffffu, ls, off);
                float zs[C::kNS];
#pragma unroll
                for (int k = 0; k < C::kNS; ++k) {
                    zs[k] = zsum[t][k][j];
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1)
                        zs[k] += __shfl_xor_sync(0xffffffffu, zs[k], off);
                }
                const int r = t * 8 + 2 * c + j;
                if (r < nq) {
                    float* dst = merge + (warp * rows + r) * C::kRecStride;
#pragma unroll
                    for (int b = 0; b < C::kSub; ++b) {
                        const float z = zs[b * 32 / BS];
                        float4 v;  // elements 32 b + 4 g + {0, 1, 2, 3}
                        v.x = fmaf(acc[t][b][0][j], 16777216.0f, z);
                        v.y = fmaf(acc[t][b][1][j], 1048576.0f, z);
                        v.z = fmaf(acc[t][b][0][j + 2], 16777216.0f, z);
                        v.w = fmaf(acc[t][b][1][j + 2], 1048576.0f, z);
                        *reinterpret_cast<float4*>(dst + 32 * b + 4 * g) = v;
                    }
                    if (g == 0) {
                        dst[D] = dead ? NAN : ls;
                        dst[D + 1] = M[t][j];
                    }
                }
            }
        __syncthreads();

        // ---- the CTA's state: thread (row, 4 elements)
        constexpr int kLanes = D / 4;
        const bool whole = walk.start >= g0 && unit_end <= g1;
        const bool starts_here = walk.start >= g0;
        for (int r = threadIdx.x / kLanes; r < nq; r += kI4Threads / kLanes) {
            const int i = threadIdx.x % kLanes;
            const float* src = merge + r * C::kRecStride;
            float m = -INFINITY;
#pragma unroll
            for (int w = 0; w < kI4Warps; ++w) m = fmaxf(m, src[w * rows * C::kRecStride + D + 1]);
            float4 v = make_float4(0, 0, 0, 0);
            float ls = 0.0f;
#pragma unroll
            for (int w = 0; w < kI4Warps; ++w) {
                const float* p = src + w * rows * C::kRecStride;
                if (p[D + 1] == -INFINITY && p[D] == 0.0f) continue;  // a warp without tiles
                const float f = fast_exp2(p[D + 1] - m);
                const float4 x = *reinterpret_cast<const float4*>(p + 4 * i);
                v.x = fmaf(x.x, f, v.x);
                v.y = fmaf(x.y, f, v.y);
                v.z = fmaf(x.z, f, v.z);
                v.w = fmaf(x.w, f, v.w);
                ls = fmaf(p[D], f, ls);
            }
            if (whole) {
                const float inv = 1.0f / ls;
                uint2 out;
                out.x = bf16 ? pack2<true>(v.x * inv, v.y * inv) : pack2<false>(v.x * inv, v.y * inv);
                out.y = bf16 ? pack2<true>(v.z * inv, v.w * inv) : pack2<false>(v.z * inv, v.w * inv);
                reinterpret_cast<uint2*>(a.o + (static_cast<long long>(walk.b) * a.Hq + head0 + r) * D)[i] = out;
            } else {
                float* rec = a.recs + ((cta * 2 + (starts_here ? 1 : 0)) * rows + r) * C::kRecStride;
                __stcg(reinterpret_cast<float4*>(rec) + i, v);
                if (i == 0) __stcg(reinterpret_cast<float2*>(rec + D), make_float2(ls, m));
            }
        }

        if (!whole) {
            // ---- the last CTA to arrive merges the unit's records
            const long long first = cta_of(walk.start), last = cta_of(unit_end - 1);
            __syncthreads();
            if (threadIdx.x == 0) {
                __threadfence();
                const unsigned int before = atomicAdd(a.counters + first, 1u);
                __threadfence();
                const bool done = before == static_cast<unsigned int>(last - first);
                if (done) a.counters[first] = 0u;
                *flag = done;
            }
            __syncthreads();
            if (*flag) {
                const long long rec_cta = 2ll * rows * C::kRecStride;
                for (int r = threadIdx.x / kLanes; r < nq; r += kI4Threads / kLanes) {
                    const int i = threadIdx.x % kLanes;
                    // the first CTA's piece is its second record, all others' the first
                    float* rec = a.recs + (first * 2 * rows + r) * C::kRecStride;
                    auto at = [&](long long p) {
                        return rec + p * rec_cta + (p == 0 ? rows * C::kRecStride : 0);
                    };
                    const int np = static_cast<int>(last - first) + 1;
                    float m = -INFINITY;
#pragma unroll 4
                    for (int p = 0; p < np; ++p) m = fmaxf(m, __ldcg(at(p) + D + 1));
                    float4 v = make_float4(0, 0, 0, 0);
                    float ls = 0.0f;
#pragma unroll 4
                    for (int p = 0; p < np; ++p) {
                        const float2 lm = __ldcg(reinterpret_cast<const float2*>(at(p) + D));
                        const float4 x = __ldcg(reinterpret_cast<const float4*>(at(p)) + i);
                        const float f = fast_exp2(lm.y - m);
                        v.x = fmaf(x.x, f, v.x);
                        v.y = fmaf(x.y, f, v.y);
                        v.z = fmaf(x.z, f, v.z);
                        v.w = fmaf(x.w, f, v.w);
                        ls = fmaf(lm.x, f, ls);
                    }
                    const float inv = 1.0f / ls;
                    uint2 out;
                    out.x = bf16 ? pack2<true>(v.x * inv, v.y * inv) : pack2<false>(v.x * inv, v.y * inv);
                    out.y = bf16 ? pack2<true>(v.z * inv, v.w * inv) : pack2<false>(v.z * inv, v.w * inv);
                    reinterpret_cast<uint2*>(a.o + (static_cast<long long>(walk.b) * a.Hq + head0 + r) * D)[i] = out;
                }
                __syncthreads();  // all reads done: the records are zero again
                for (long long p = first; p <= last; ++p) {
                    float4* rec = reinterpret_cast<float4*>(
                        a.recs + (p * 2 + (p == first ? 1 : 0)) * rows * C::kRecStride);
                    for (int i = threadIdx.x; i < nq * C::kRecStride / 4; i += kI4Threads)
                        __stcg(rec + i, make_float4(0, 0, 0, 0));
                }
            }
        }
        __syncthreads();  // the merge area and the flag are free again
        p0 = p1;
    }
}

}  // namespace tqkv
