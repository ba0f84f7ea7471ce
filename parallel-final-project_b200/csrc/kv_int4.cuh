// kv_int4.cuh — the 4-bit KV cache: quantising rows as they are written,
// reading them back, and the head norms with the position rotation that
// produce the rows, for sm_100a.
//
// Format.  A row of D elements has D / BS blocks.  Per block, all arithmetic
// in fp32 with IEEE rounding:
//     zero  = fp16(min x)
//     scale = fp16((max x - min x) / 15)
//     code  = clamp(round_half_even((x - zero) / scale), 0, 15); 0 if scale = 0
//     value = code * scale + zero
// A block whose scale or zero is not finite (an input that is NaN, infinite or
// outside fp16's range) gets scale = zero = NaN and codes 0: it reads back as
// NaN instead of as a plausible number.
//
// Packed order.  A row is D / 8 32-bit words of eight codes, the first code in
// the lowest bits.  Elements 8 l .. 8 l + 7 are word (l % 4) * (D / 32) + l / 4:
// the four words of a 32-element group lie D / 8 bytes apart.  So the 16 bytes
// (8 for D = 64) at offset c * D / 8 hold one word of every 32-element group,
// and a decode lane that loads them with one instruction can still apply a
// scale per group (decode_int4.cuh).
//
// Bound: HBM.  One lane owns 8 elements (one 16-byte load), D / 8 lanes a row.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "device_common.cuh"
#include "kv_compress.cuh"

namespace tqkv {

// n / d and n % d for n < 2^31 by one multiplication (Granlund and
// Montgomery, 1994): q = (mulhi(n, m) + n) >> s with 2^s >= d.
struct FastDiv {
    uint32_t d, m, s;
    FastDiv() = default;
    explicit FastDiv(uint32_t d_) : d(d_), m(0), s(0) {
        while ((1ull << s) < d) ++s;
        m = static_cast<uint32_t>(((1ull << 32) * ((1ull << s) - d)) / d + 1);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const {
        return (__umulhi(n, m) + n) >> s;
    }
};

// max / min that keep a NaN operand
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <bool BF16>
__device__ __forceinline__ void unpack8(uint4 raw, float (&f)[8]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (BF16) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            f[2 * i] = v.x;
            f[2 * i + 1] = v.y;
        }
    }
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}

// Codes of one lane's 8 values, given its block's minimum and maximum; sets
// `params` to the block's (scale, zero).
//
// The quotient d / scale decides a code by its distance from a half-integer,
// and fp16 inputs do meet half-integers exactly, where a reciprocal rounded to
// 24 bits would fall to either side.  So the reciprocal is carried in two
// words, r + e with e = (1 - scale * r) * r: d * r + d * e has a relative
// error below 2^-45 before its one rounding, which returns an exact
// half-integer quotient as that half-integer.  One multiply and one FMA an
// element instead of a division.
__device__ __forceinline__ uint32_t int4_codes(const float (&f)[8], float lo, float hi,
                                               uint32_t& params) {
    __half zero = __float2half_rn(lo);
    __half scale = __float2half_rn(__fdiv_rn(hi - lo, 15.0f));
    float z = __half2float(zero);
    float s = __half2float(scale);
    float r = 0.0f, e = 0.0f;
    if (!(fabsf(s) < INFINITY && fabsf(z) < INFINITY)) {
        zero = scale = __ushort_as_half(0x7fff);
    } else if (s > 0.0f) {
        r = __frcp_rn(s);
        e = fmaf(-s, r, 1.0f) * r;
    }
    params = __half_as_ushort(scale) | (static_cast<uint32_t>(__half_as_ushort(zero)) << 16);
    // 1.5 * 2^23 + q rounds q to an integer, ties to even, in the low bits;
    // fmaxf(NaN, 0) = 0 covers the blocks with r = 0 and infinite elements
    constexpr float kMagic = 12582912.0f;
    uint32_t word = 0;
#pragma unroll
    for (int i = 7; i >= 0; --i) {
        const float d = f[i] - z;
        const float q = fminf(fmaxf(fmaf(d, r, d * e), 0.0f), 15.0f);
        word = (word << 4) | (__float_as_uint(q + kMagic) & 15u);
    }
    return word;
}

// Minimum and maximum over the lane's block (aligned groups of BS / 8 lanes).
template <int BS>
__device__ __forceinline__ void block_range(const float (&f)[8], float& lo, float& hi) {
    lo = hi = f[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        lo = min_nan(lo, f[i]);
        hi = max_nan(hi, f[i]);
    }
#pragma unroll
    for (int off = 1; off < BS / 8; off <<= 1) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, off));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, off));
    }
}

// Where lane l's word stands in a packed row.
template <int D>
__device__ __forceinline__ int word_of_lane(int l) {
    return (l & 3) * (D / 32) + (l >> 2);
}

// Quantises lane l's 8 values of a row into the cache row `row`.  Every lane
// of the warp calls it; rows with `valid` false are computed and dropped.
template <int D, int BS>
__device__ __forceinline__ void store_int4(const float (&f)[8], int l, long long row, bool valid,
                                           uint32_t* __restrict__ codes,
                                           uint32_t* __restrict__ params) {
    float lo, hi;
    block_range<BS>(f, lo, hi);
    uint32_t p;
    const uint32_t w = int4_codes(f, lo, hi, p);
    if (!valid) return;
    codes[row * (D / 8) + word_of_lane<D>(l)] = w;
    if (l % (BS / 8) == 0) params[row * (D / BS) + l / (BS / 8)] = p;
}

// Rows [start_b, start_b + T) of every head of a cache, or of x.
struct Int4Rows {
    uint32_t rows;          // B * H * T
    FastDiv T, H;
    long long S_cap;
    const int32_t* starts;  // [B], or null: t0 for every sequence
    int t0;
    long long sb, sh, st;   // strides of x in elements (kv_append)

    // row r = (b * H + h) * T + t: sets its place in the cache and in x;
    // false if that row of the cache does not exist
    __device__ __forceinline__ bool locate(uint32_t r, long long& cache_row,
                                           long long& x_off) const {
        const uint32_t bh = T.div(r);
        const uint32_t t = r - bh * T.d;
        const uint32_t b = H.div(bh);
        const long long pos = static_cast<long long>(starts ? starts[b] : t0) + t;
        cache_row = static_cast<long long>(bh) * S_cap + pos;
        x_off = b * sb + (bh - b * H.d) * sh + t * st;
        return pos >= 0 && pos < S_cap;
    }
};

constexpr int kInt4Threads = 256;
constexpr int kInt4Unroll = 4;  // rows a lane keeps in flight

template <int D, int BS, bool BF16>
__global__ void __launch_bounds__(kInt4Threads)
    kv_append_int4_kernel(const uint16_t* __restrict__ x, uint32_t* __restrict__ codes,
                          uint32_t* __restrict__ params, Int4Rows g) {
    griddep_wait();
    griddep_launch_dependents();
    constexpr int kLPR = D / 8;
    constexpr int kRPW = 32 / kLPR;
    const int l = (threadIdx.x & 31) % kLPR;
    const uint32_t warp = (blockIdx.x * kInt4Threads + threadIdx.x) >> 5;
    const uint32_t r0 = warp * (kRPW * kInt4Unroll) + (threadIdx.x & 31) / kLPR;
    long long row[kInt4Unroll];
    bool ok[kInt4Unroll];
    uint4 raw[kInt4Unroll];
#pragma unroll
    for (int u = 0; u < kInt4Unroll; ++u) {
        const uint32_t r = r0 + u * kRPW;
        long long off = 0;
        row[u] = 0;
        ok[u] = r < g.rows && g.locate(r, row[u], off);
        raw[u] = make_uint4(0, 0, 0, 0);
        if (ok[u]) raw[u] = ld_stream_v4(reinterpret_cast<const uint4*>(x + off) + l);
    }
#pragma unroll
    for (int u = 0; u < kInt4Unroll; ++u) {
        float f[8];
        unpack8<BF16>(raw[u], f);
        store_int4<D, BS>(f, l, row[u], ok[u], codes, params);
    }
}

// Eight values of one packed word.  code * scale + zero is rounded once to
// fp16 by a half-precision FMA (codes are exact in fp16); for bf16 the sum is
// formed in fp32 and rounded to bf16.
template <bool BF16>
__device__ __forceinline__ uint4 int4_values(uint32_t w, uint32_t params) {
    const __half2 p = *reinterpret_cast<const __half2*>(&params);
    const __half2 s2 = __low2half2(p), z2 = __high2half2(p);
    // 0x6400 | nibble is 1024 + nibble; the nibble in bits 4..7 is 1024 + 16 n
    const __half2 k1024 = __half2half2(__ushort_as_half(0x6400));
    const __half2 k1024over16 = __half2half2(__ushort_as_half(0xd400));  // -64
    const __half2 k16th = __half2half2(__ushort_as_half(0x2c00));        // 1 / 16
    __half2 n04, n15, n26, n37;
    {
        const uint32_t a = (w & 0x000f000fu) | 0x64006400u, b = (w & 0x00f000f0u) | 0x64006400u;
        const uint32_t v = w >> 8;
        const uint32_t c = (v & 0x000f000fu) | 0x64006400u, d = (v & 0x00f000f0u) | 0x64006400u;
        n04 = __hsub2_rn(*reinterpret_cast<const __half2*>(&a), k1024);
        n26 = __hsub2_rn(*reinterpret_cast<const __half2*>(&c), k1024);
        n15 = __hfma2(*reinterpret_cast<const __half2*>(&b), k16th, k1024over16);
        n37 = __hfma2(*reinterpret_cast<const __half2*>(&d), k16th, k1024over16);
    }
    const __half2 n[4] = {__lows2half2(n04, n15), __lows2half2(n26, n37),
                          __highs2half2(n04, n15), __highs2half2(n26, n37)};
    uint32_t out[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (BF16) {
            const float2 c = __half22float2(n[i]);
            const float s = __low2float(p), z = __high2float(p);
            out[i] = pack2<true>(fmaf(c.x, s, z), fmaf(c.y, s, z));
        } else {
            const __half2 v = __hfma2(n[i], s2, z2);
            out[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
    return make_uint4(out[0], out[1], out[2], out[3]);
}

// y[r] = the values of the cache's row; rows that the cache does not have
// read as zero.
template <int D, int BS, bool BF16>
__global__ void __launch_bounds__(kInt4Threads)
    kv_reconstruct_int4_kernel(const uint32_t* __restrict__ codes,
                               const uint32_t* __restrict__ params, uint4* __restrict__ y,
                               Int4Rows g) {
    griddep_wait();
    griddep_launch_dependents();
    constexpr int kLPR = D / 8;
    constexpr int kRPW = 32 / kLPR;
    const int l = (threadIdx.x & 31) % kLPR;
    const uint32_t warp = (blockIdx.x * kInt4Threads + threadIdx.x) >> 5;
    const uint32_t r0 = warp * (kRPW * kInt4Unroll) + (threadIdx.x & 31) / kLPR;
    uint32_t w[kInt4Unroll], p[kInt4Unroll];
#pragma unroll
    for (int u = 0; u < kInt4Unroll; ++u) {
        const uint32_t r = r0 + u * kRPW;
        long long row = 0, off = 0;
        w[u] = p[u] = 0;
        if (r < g.rows && g.locate(r, row, off)) {
            w[u] = codes[row * (D / 8) + word_of_lane<D>(l)];
            p[u] = params[row * (D / BS) + l / (BS / 8)];
        }
    }
#pragma unroll
    for (int u = 0; u < kInt4Unroll; ++u) {
        const uint32_t r = r0 + u * kRPW;
        if (r < g.rows)
            st_stream_v4(y + static_cast<long long>(r) * kLPR + l, int4_values<BF16>(w[u], p[u]));
    }
}

// ---------------------------------------------------------------------------
// Head norms and position rotation
//
//   y   = x * rsqrt(mean x^2 + eps) * w          per head, over its D elements
//   out = (a cos - b sin, b cos + a sin)         for each pair (a, b) of y
//
// with pair j = elements (j, j + rot / 2), or (2 j, 2 j + 1) interleaved, and
// (cos, sin) from column j of a table's row; the row is the token's position
// on the axis that pair j belongs to.  K rows can go straight into the 4-bit
// cache, and V rows with them.
//
// The values decide 4-bit codes, where a difference in the last bit can move
// a code, so they do not depend on the order of a sum: the mean square is
// summed in fp64 (squares of 16-bit inputs lose nothing that fp32 would show)
// and its reciprocal root is the fp64 one rounded to fp32; the products and
// sums after it are rounded one by one (no contraction).
//
// A row is D / 16 lanes; a lane holds two runs of 8 elements such that the
// halves of a pair meet in one lane (elements 8 l .. and rot / 2 + 8 l ..), so
// the rotation needs no other lane, and 8 elements are one word of the 4-bit
// format.  A lane group takes one token and up to heads_per_group heads of one
// kind, so that the table's 64 bytes a lane (against 32 of data) are read once
// for those heads.
struct RopeArgs {
    const uint16_t *q, *k, *v;     // element (b, h, t, 0) at b * sb + h * sh + t * st
    long long q_sb, q_sh, q_st, k_sb, k_sh, k_st, v_sb, v_sh, v_st;
    uint16_t *q_out, *k_out;       // [B, H, T, D]
    const uint16_t *q_w, *k_w;     // [D] or null
    const float2* table;           // [max_pos, rot / 2]
    const int32_t* pos;            // [axes, B, T]
    uint32_t *kc, *kp, *vc, *vp;   // 4-bit caches (append)
    const int32_t* starts;         // [B] or null
    double eps;
    long long S_cap;
    uint32_t tokens;               // B * T
    int Hq, Hkv, T, t0, max_pos, rot, heads_per_group;
    int q_groups, kv_groups;       // lane groups a token needs for q, and for k (and for v)
    int s1, s2, s3;                // first pair of axes 1, 2, 3
    int axes;
    FastDiv groups, divT;          // lane groups a token needs in all
};

// 1 / sqrt(x) rounded to fp32 as if from its exact value: one Newton step in
// fp64 from the fp32 approximation (relative error 2^-22, then 2^-43).
__device__ __forceinline__ float rsqrt_rounded(double x) {
    if (!(x > 1e-36 && x < 1e36)) return static_cast<float>(rsqrt(x));
    const double y = rsqrtf(static_cast<float>(x));
    return static_cast<float>(fma(0.5 * y, fma(-x * y, y, 1.0), y));
}

// Minimum and maximum of lane runs over blocks of BS elements, 8 a lane:
// aligned groups of BS / 8 lanes when `a` and `b` are different blocks, or, for
// BS = D, both runs of every lane of the row.
template <int D, int BS>
__device__ __forceinline__ void store_int4_runs(const float (&a)[8], const float (&b)[8], int l,
                                                long long row, bool valid,
                                                uint32_t* __restrict__ codes,
                                                uint32_t* __restrict__ params) {
    constexpr int kLanes = D / 16;  // lanes a row has; run a is element 8 l, run b D / 2 + 8 l
    float lo[2] = {a[0], b[0]}, hi[2] = {a[0], b[0]};
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        lo[0] = min_nan(lo[0], a[i]);
        hi[0] = max_nan(hi[0], a[i]);
        lo[1] = min_nan(lo[1], b[i]);
        hi[1] = max_nan(hi[1], b[i]);
    }
    if constexpr (BS == D) {
        lo[0] = lo[1] = min_nan(lo[0], lo[1]);
        hi[0] = hi[1] = max_nan(hi[0], hi[1]);
    }
    constexpr int kGroup = BS == D ? kLanes : BS / 8;
#pragma unroll
    for (int h = 0; h < (BS == D ? 1 : 2); ++h)
#pragma unroll
        for (int off = 1; off < kGroup; off <<= 1) {
            lo[h] = min_nan(lo[h], __shfl_xor_sync(0xffffffffu, lo[h], off));
            hi[h] = max_nan(hi[h], __shfl_xor_sync(0xffffffffu, hi[h], off));
        }
    if constexpr (BS == D) lo[1] = lo[0], hi[1] = hi[0];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t p;
        const uint32_t w = int4_codes(h == 0 ? a : b, lo[h], hi[h], p);
        if (!valid) continue;
        const int run = l + h * kLanes;
        codes[row * (D / 8) + word_of_lane<D>(run)] = w;
        if (run % (BS / 8) == 0) params[row * (D / BS) + run / (BS / 8)] = p;
    }
}

constexpr int kRopeUnroll = 2;  // heads whose rows a lane group has in flight

template <int D, int BS, bool BF16, bool APPEND, bool INTERLEAVED>
__global__ void __launch_bounds__(kInt4Threads, 2) qk_norm_rope_kernel(const RopeArgs a) {
    griddep_wait();
    griddep_launch_dependents();
    constexpr int kLanes = D / 16;
    const int lane = threadIdx.x & 31;
    const int l = lane % kLanes;
    const uint32_t unit = (blockIdx.x * kInt4Threads + threadIdx.x) / kLanes;
    uint32_t tok = a.groups.div(unit);
    int grp = static_cast<int>(unit - tok * a.groups.d);
    const bool live = tok < a.tokens;
    if (!live) tok = 0, grp = 0;   // keeps the warp's shuffles whole; stores nothing
    const uint32_t b = a.divT.div(tok);
    const uint32_t t = tok - b * a.divT.d;

    int kind = 0;  // 0: q, 1: k, 2: v
    if (grp >= a.q_groups) {
        grp -= a.q_groups;
        kind = 1;
        if (grp >= a.kv_groups) grp -= a.kv_groups, kind = 2;
    }
    const int h0 = grp * a.heads_per_group;
    const int H = kind == 0 ? a.Hq : a.Hkv;
    const int h1 = h0 + a.heads_per_group < H ? h0 + a.heads_per_group : H;
    const uint16_t* x = kind == 0 ? a.q + b * a.q_sb + t * a.q_st
                        : kind == 1 ? a.k + b * a.k_sb + t * a.k_st
                                    : a.v + b * a.v_sb + t * a.v_st;
    const long long sh = kind == 0 ? a.q_sh : kind == 1 ? a.k_sh : a.v_sh;

    // runs (in units of 8 elements): the pairs' halves of the rotated part, and
    // the halves of what is behind it
    const int rot_lanes = a.rot / 16;
    const bool rotates = l < rot_lanes && kind != 2;
    const bool natural = INTERLEAVED || a.rot == D || kind == 2;  // runs l and l + kLanes
    const int run0 = natural || l < rot_lanes ? l : rot_lanes + l;
    const int run1 = natural ? l + kLanes : l < rot_lanes ? rot_lanes + l : kLanes + l;
    float2 cs[8];
    bool turns[2] = {rotates, rotates};  // interleaved: whether run 0 and run 1 rotate
    if (INTERLEAVED) {
        turns[0] = kind != 2 && run0 < 2 * rot_lanes;
        turns[1] = kind != 2 && run1 < 2 * rot_lanes;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int j = INTERLEAVED ? (i < 4 ? run0 : run1) * 4 + (i & 3) : l * 8 + i;
        cs[i] = make_float2(1.0f, 0.0f);
        if (turns[INTERLEAVED ? i >> 2 : 0]) {
            const int axis = a.axes == 1 ? 0 : (j >= a.s1) + (j >= a.s2) + (j >= a.s3);
            const int p = a.pos[static_cast<long long>(axis) * a.tokens + tok];
            // a position outside the table leaves NaN in the row
            cs[i] = p >= 0 && p < a.max_pos
                        ? a.table[static_cast<long long>(p) * (a.rot / 2) + j]
                        : make_float2(NAN, NAN);
        }
    }
    const uint16_t* wsrc = kind == 0 ? a.q_w : kind == 1 ? a.k_w : nullptr;
    float w0[8], w1[8];
    if (wsrc) {
        unpack8<BF16>(reinterpret_cast<const uint4*>(wsrc)[run0], w0);
        unpack8<BF16>(reinterpret_cast<const uint4*>(wsrc)[run1], w1);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) w0[i] = w1[i] = 1.0f;
    }

    const bool norms = __any_sync(0xffffffffu, kind != 2);   // some row of the warp is q's or k's
    const bool caches = __any_sync(0xffffffffu, kind != 0);  // some row goes to a cache, if any does
    for (int hb = h0; __any_sync(0xffffffffu, hb < h1); hb += kRopeUnroll) {
        uint4 raw[kRopeUnroll][2];
#pragma unroll
        for (int u = 0; u < kRopeUnroll; ++u) {
            raw[u][0] = raw[u][1] = make_uint4(0, 0, 0, 0);
            if (hb + u < h1) {
                const uint4* src = reinterpret_cast<const uint4*>(x + (hb + u) * sh);
                raw[u][0] = src[run0];
                raw[u][1] = src[run1];
            }
        }
#pragma unroll
        for (int u = 0; u < kRopeUnroll; ++u) {
            const int h = hb + u;
            if (!__any_sync(0xffffffffu, h < h1)) break;
            float f0[8], f1[8];
            unpack8<BF16>(raw[u][0], f0);
            unpack8<BF16>(raw[u][1], f1);
            if (norms) {
                double ss = 0.0, st = 0.0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const double p = f0[i], q = f1[i];
                    ss = fma(p, p, ss);
                    st = fma(q, q, st);
                }
                ss += st;
#pragma unroll
                for (int off = 1; off < kLanes; off <<= 1)
                    ss += __shfl_xor_sync(0xffffffffu, ss, off);
                if (kind != 2) {
                    const float inv = rsqrt_rounded(ss * (1.0 / D) + a.eps);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        f0[i] = __fmul_rn(__fmul_rn(f0[i], inv), w0[i]);
                        f1[i] = __fmul_rn(__fmul_rn(f1[i], inv), w1[i]);
                    }
                    if constexpr (INTERLEAVED) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            float* f = i < 4 ? f0 + 2 * i : f1 + 2 * (i - 4);
                            if (!turns[i >> 2]) continue;
                            const float p = f[0], q = f[1];
                            f[0] = __fsub_rn(__fmul_rn(p, cs[i].x), __fmul_rn(q, cs[i].y));
                            f[1] = __fadd_rn(__fmul_rn(q, cs[i].x), __fmul_rn(p, cs[i].y));
                        }
                    } else if (rotates) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float p = f0[i], q = f1[i];
                            f0[i] = __fsub_rn(__fmul_rn(p, cs[i].x), __fmul_rn(q, cs[i].y));
                            f1[i] = __fadd_rn(__fmul_rn(q, cs[i].x), __fmul_rn(p, cs[i].y));
                        }
                    }
                }
            }
            const bool store = live && h < h1;
            if (!APPEND || kind == 0) {
                if (store) {
                    uint16_t* out = kind == 0 ? a.q_out : a.k_out;
                    const long long row = (static_cast<long long>(b) * H + h) * a.T + t;
                    uint4* dst = reinterpret_cast<uint4*>(out) + row * (D / 8);
                    dst[run0] = make_uint4(pack2<BF16>(f0[0], f0[1]), pack2<BF16>(f0[2], f0[3]),
                                           pack2<BF16>(f0[4], f0[5]), pack2<BF16>(f0[6], f0[7]));
                    dst[run1] = make_uint4(pack2<BF16>(f1[0], f1[1]), pack2<BF16>(f1[2], f1[3]),
                                           pack2<BF16>(f1[4], f1[5]), pack2<BF16>(f1[6], f1[7]));
                }
            }
            if constexpr (APPEND) {
                if (!caches) continue;
                if (!INTERLEAVED && a.rot != D) {
                    // runs back into their natural order: run r is in lane `from`, first or second
                    float n0[8], n1[8];
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        const int r = l + s * kLanes;
                        int from = r;
                        bool is_second = r >= kLanes;
                        if (kind != 2) {
                            const int tail = kLanes - rot_lanes;  // lanes behind the rotated part
                            is_second = r < 2 * rot_lanes ? r >= rot_lanes : r - 2 * rot_lanes >= tail;
                            from = r < 2 * rot_lanes ? (is_second ? r - rot_lanes : r)
                                                     : r - rot_lanes - (is_second ? tail : 0);
                        } else if (is_second) {
                            from = r - kLanes;
                        }
                        from += lane - l;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float p = __shfl_sync(0xffffffffu, f0[i], from);
                            const float q = __shfl_sync(0xffffffffu, f1[i], from);
                            (s == 0 ? n0 : n1)[i] = is_second ? q : p;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) f0[i] = n0[i], f1[i] = n1[i];
                }
                // lanes of q rows take part in the shuffles and store nothing
                const long long pos =
                    static_cast<long long>(a.starts ? a.starts[b] : a.t0) + static_cast<int>(t);
                const bool ok = store && kind != 0 && pos >= 0 && pos < a.S_cap;
                const long long row = (static_cast<long long>(b) * a.Hkv + h) * a.S_cap + pos;
                store_int4_runs<D, BS>(f0, f1, l, row, ok, kind == 1 ? a.kc : a.vc,
                                       kind == 1 ? a.kp : a.vp);
            }
        }
    }
}

}  // namespace tqkv
