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
// Bound: HBM, with the issue slots close behind; so a lane owns 16 elements,
// D / 16 lanes a row, which halves what every lane does once per row and block.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>

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

// `bytes` (4, 8 or 16) of global memory into shared memory, or zeros
template <int bytes>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, bool real = true) {
    if constexpr (bytes == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
                     "r"(real ? 16 : 0)
                     : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src),
                     "n"(bytes), "r"(real ? bytes : 0)
                     : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

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

// What a block's codes are made with.
struct BlockScale {
    float zero, r, e;  // 1 / (16 scale) = r + e
    uint32_t params;   // (scale, zero) as stored
};

// The quotient d / scale decides a code by its distance from a half-integer,
// and fp16 inputs do meet half-integers exactly, where a reciprocal rounded to
// 24 bits would fall to either side.  So the reciprocal is carried in two
// words, r + e with e = (1 - scale * r) * r: d * r + d * e has a relative
// error below 2^-43 before its one rounding, which returns an exact
// half-integer quotient as that half-integer.  One multiply and one FMA an
// element instead of a division.  The range's fifteenth likewise: a product with
// 1 / 15 rounded to 24 bits moves every quotient a little up, and of those that lie
// between two fp16 values (ranges of 15 odd multiples of half a step) 439 of 1024 to the
// wrong one.  With 1 / 15 in two words the product is off by less than 2^-46 before its
// one rounding, and a quotient by 15 lies at least 1 / 30 of a step from the middle
// between two fp32 values: it is the division's.
__device__ __forceinline__ BlockScale block_scale(float lo, float hi) {
    constexpr float k15 = 1.0f / 15.0f;
    constexpr float k15low = static_cast<float>(1.0 / 15.0 - static_cast<double>(k15));
    const float range = hi - lo;
    __half zero = __float2half_rn(lo);
    __half scale = __float2half_rn(fmaf(range, k15, range * k15low));
    const float s = __half2float(scale);
    BlockScale b;
    b.zero = __half2float(zero);
    b.r = b.e = 0.0f;
    if (!(fabsf(s) < INFINITY && fabsf(b.zero) < INFINITY)) {
        zero = scale = __ushort_as_half(0x7fff);
    } else if (s > 0.0f) {
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(b.r) : "f"(s));
        b.e = fmaf(-s, b.r, 1.0f) * b.r * 0.0625f;
        b.r *= 0.0625f;
    }
    b.params = __half_as_ushort(scale) | (static_cast<uint32_t>(__half_as_ushort(zero)) << 16);
    return b;
}

// One word of codes.  A quotient over 16 is clamped to [0, 1] by the FMA's
// saturation, which also turns NaN to 0 (a block with r = 0 whose elements are
// infinite), and to 15 / 16; 1.5 * 2^23 + 16 t then rounds it to an integer,
// ties to even, in the low bits.  The words' sum of 16^i times those floats'
// bits differs from the codes' by a constant.
__device__ __forceinline__ uint32_t int4_codes(const float* f, const BlockScale& b) {
    constexpr float kMagic = 12582912.0f;  // bits 0x4b400000
    uint32_t word = 0;
#pragma unroll
    for (int i = 7; i >= 0; --i) {
        const float d = f[i] - b.zero;
        const float t = fminf(__saturatef(fmaf(d, b.r, d * b.e)), 0.9375f);
        word = word * 16u + __float_as_uint(fmaf(t, 16.0f, kMagic));
    }
    return word - 0x4b400000u * 0x11111111u;
}

// Where lane l's word stands in a packed row.
template <int D>
__device__ __forceinline__ int word_of_lane(int l) {
    return (l & 3) * (D / 32) + (l >> 2);
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

// Small CTAs with little work a lane: 17.5 us for writing and reading back 131,072
// rows of 128 in two launches, 18.4 with 256 threads and twice the rows a lane;
// 3.5 and 4.6 us for one row of each of 512 heads.  One row a lane when reading
// back shortens that to 3.0, but a long cache takes 136 us instead of 102.
constexpr int kInt4Threads = 128;
constexpr int kReadUnroll = 2;  // rows a lane has in flight when it reads back

// Packed maximum of 16-bit pairs, NaN if either is.
template <bool BF16>
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
    if constexpr (BF16) {
        const __nv_bfloat162 v = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                             *reinterpret_cast<const __nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __half2 v = __hmax2_nan(*reinterpret_cast<const __half2*>(&a),
                                      *reinterpret_cast<const __half2*>(&b));
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}

template <bool BF16>
__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b) {
    if constexpr (BF16) {
        const __nv_bfloat162 v = __hmin2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                             *reinterpret_cast<const __nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __half2 v = __hmin2_nan(*reinterpret_cast<const __half2*>(&a),
                                      *reinterpret_cast<const __half2*>(&b));
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}

// Range of the block that the lane's 16 elements belong to (aligned groups of
// BS / 16 lanes): maximum and negated minimum go through one reduction.
template <int BS, bool BF16>
__device__ __forceinline__ void block_range16(const uint32_t (&w)[8], float& lo, float& hi) {
    uint32_t mx = w[0], mn = w[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        mx = max2_nan<BF16>(mx, w[i]);
        mn = min2_nan<BF16>(mn, w[i]);
    }
    mn ^= 0x80008000u;
    // (largest of the even, negated smallest of the even) and the same of the odd elements
    uint32_t m = max2_nan<BF16>(__byte_perm(mx, mn, 0x5410), __byte_perm(mx, mn, 0x7632));
#pragma unroll
    for (int off = 1; off < BS / 16; off <<= 1)
        m = max2_nan<BF16>(m, __shfl_xor_sync(0xffffffffu, m, off));
    if constexpr (BF16) {
        hi = __uint_as_float(m << 16);
        lo = -__uint_as_float(m & 0xffff0000u);
    } else {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&m));
        hi = v.x;
        lo = -v.y;
    }
}

template <int D, int BS, bool BF16>
__global__ void __launch_bounds__(kInt4Threads)
    kv_append_int4_kernel(const uint16_t* __restrict__ x, uint32_t* __restrict__ codes,
                          uint32_t* __restrict__ params, const Int4Rows g) {
    griddep_wait();
    griddep_launch_dependents();
    constexpr int kLanes = D / 16;
    const int l = threadIdx.x % kLanes;
    const uint32_t r = blockIdx.x * (kInt4Threads / kLanes) + threadIdx.x / kLanes;
    long long row = 0, off = 0;
    const bool ok = r < g.rows && g.locate(r, row, off);
    uint4 a = make_uint4(0, 0, 0, 0), b = a;
    if (ok) {
        a = reinterpret_cast<const uint4*>(x + off)[2 * l];
        b = reinterpret_cast<const uint4*>(x + off)[2 * l + 1];
    }
    const uint32_t raw[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    float lo, hi;
    block_range16<BS, BF16>(raw, lo, hi);
    if (!ok) return;
    const BlockScale scale = block_scale(lo, hi);
    // runs 2 l and 2 l + 1 are neighbours of one 32-element group
    uint32_t* dst = codes + row * (D / 8) + word_of_lane<D>(2 * l);
    float f[8];
    unpack8<BF16>(a, f);
    dst[0] = int4_codes(f, scale);
    unpack8<BF16>(b, f);
    dst[D / 32] = int4_codes(f, scale);
    if (l % (BS / 16) == 0) params[row * (D / BS) + l / (BS / 16)] = scale.params;
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
// read as zero.  A lane takes runs of 8 elements r and r + 4, whose words are
// neighbours: 8 bytes in, twice 16 out.
template <int D, int BS, bool BF16>
__global__ void __launch_bounds__(kInt4Threads)
    kv_reconstruct_int4_kernel(const uint32_t* __restrict__ codes,
                               const uint32_t* __restrict__ params, uint4* __restrict__ y,
                               const Int4Rows g) {
    griddep_wait();
    griddep_launch_dependents();
    constexpr int kLanes = D / 16;
    constexpr int kRPW = 32 / kLanes;
    const int l = (threadIdx.x & 31) % kLanes;
    const int run = l % 4 + 8 * (l / 4);
    const uint32_t warp = blockIdx.x * (kInt4Threads / 32) + threadIdx.x / 32;
    const uint32_t r0 = warp * (kRPW * kReadUnroll) + (threadIdx.x & 31) / kLanes;
    uint2 w[kReadUnroll], p[kReadUnroll];
#pragma unroll
    for (int u = 0; u < kReadUnroll; ++u) {
        const uint32_t r = r0 + u * kRPW;
        long long row = 0, off = 0;
        w[u] = p[u] = make_uint2(0, 0);
        if (r < g.rows && g.locate(r, row, off)) {
            w[u] = *reinterpret_cast<const uint2*>(codes + row * (D / 8) + word_of_lane<D>(run));
            if constexpr (BS == 32) {
                p[u] = *reinterpret_cast<const uint2*>(params + row * (D / BS) + run / 4);
            } else {
                p[u].x = params[row * (D / BS) + run / (BS / 8)];
                p[u].y = p[u].x;
            }
        }
    }
#pragma unroll
    for (int u = 0; u < kReadUnroll; ++u) {
        const uint32_t r = r0 + u * kRPW;
        if (r < g.rows) {
            uint4* dst = y + static_cast<long long>(r) * (D / 8) + run;
            st_stream_v4(dst, int4_values<BF16>(w[u].x, p[u].x));
            st_stream_v4(dst + 4, int4_values<BF16>(w[u].y, p[u].y));
        }
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
// Values that go to the cache decide 4-bit codes, where a difference in the
// last bit can move a code, so there (APPEND) they do not depend on the order
// of a sum: the mean square is summed in fp64 and its reciprocal root is the
// fp64 one rounded to fp32; the products and sums after it are rounded one by
// one.  Without a cache all of it is fp32 with FMAs: fp64 and the separate
// roundings add 4 us to the 33 that 8194 tokens x 40 heads of 128 take.
//
// A row is D / 16 lanes; a lane holds two runs of 8 elements such that the
// halves of a pair meet in one lane (elements 8 l .. and rot / 2 + 8 l ..), so
// the rotation needs no other lane, and 8 elements are one word of the 4-bit
// format.  A warp takes one token and goes over its q, k and v heads, 512 / D
// side by side, so that the table's 64 bytes a lane (against 32 of data a
// head) are read once for them.  All tokens' steps, end to end, are cut into
// equal runs, one a resident warp.
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
    int Hq, Hkv, T, t0, max_pos, rot;
    int q_steps, kv_steps;         // steps of 512 / D heads: of q, of k (and of v)
    uint32_t warps, run, longer;   // a warp takes `run` steps, the first `longer` one more
    int s1, s2, s3;                // first pair of axes 1, 2, 3
    int axes;
    FastDiv steps, divT;           // steps of a token
};

// 1 / sqrt(x) rounded to fp32 as if from its exact value: one Newton step in
// fp64 from the fp32 approximation (relative error 2^-22, then 2^-43).
__device__ __forceinline__ float rsqrt_rounded(double x) {
    if (!(x > 1e-36 && x < 1e36)) return static_cast<float>(rsqrt(x));
    const double y = rsqrtf(static_cast<float>(x));
    return static_cast<float>(fma(0.5 * y, fma(-x * y, y, 1.0), y));
}

// Reciprocal root mean square of a row of D / 16 lanes, 16 elements each.
template <int D>
__device__ __forceinline__ float inv_rms_exact(const float (&a)[8], const float (&b)[8], double eps) {
    double s = 0.0, t = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const double p = a[i], q = b[i];
        s = fma(p, p, s);
        t = fma(q, q, t);
    }
    s += t;
#pragma unroll
    for (int off = 1; off < D / 16; off <<= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    return rsqrt_rounded(s * (1.0 / D) + eps);
}

// The same in fp32; rows whose squares leave fp32's range take the fp64 way, each for itself: a row's
// bits depend neither on the rows beside it nor on what stands where a row does not exist.
template <int D>
__device__ __forceinline__ float inv_rms(const float (&a)[8], const float (&b)[8], double eps, bool exists) {
    float s = 0.0f, t = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        s = fmaf(a[i], a[i], s);
        t = fmaf(b[i], b[i], t);
    }
    s += t;
#pragma unroll
    for (int off = 1; off < D / 16; off <<= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    const bool outside = exists && !(s > 1e-30f && s < 1e38f);
    float inv = __frsqrt_rn(fmaf(s, 1.0f / D, static_cast<float>(eps)));
    if (__any_sync(0xffffffffu, outside)) {  // all lanes, for the shuffles
        const float wide = inv_rms_exact<D>(a, b, eps);
        if (outside) inv = wide;
    }
    return inv;
}

// (p cos - q sin, q cos + p sin), every operation rounded by itself (EXACT) or with FMAs
template <bool EXACT>
__device__ __forceinline__ void rotate_pair(const float p, const float q, float2 cs, float& u, float& v) {
    if constexpr (EXACT) {
        u = __fsub_rn(__fmul_rn(p, cs.x), __fmul_rn(q, cs.y));
        v = __fadd_rn(__fmul_rn(q, cs.x), __fmul_rn(p, cs.y));
    } else {
        u = fmaf(p, cs.x, -(q * cs.y));
        v = fmaf(q, cs.x, p * cs.y);
    }
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
        const BlockScale s = block_scale(lo[h], hi[h]);
        const uint32_t w = int4_codes(h == 0 ? a : b, s);
        if (!valid) continue;
        const int run = l + h * kLanes;
        codes[row * (D / 8) + word_of_lane<D>(run)] = w;
        if (run % (BS / 8) == 0) params[row * (D / BS) + run / (BS / 8)] = s.params;
    }
}

constexpr int kRopeCtas = 4;   // resident on an SM
constexpr int kRopeDepth = 4;  // 1 KB a warp and step: 64 KB of an SM's 16 warps in flight

template <int D, int BS, bool BF16, bool APPEND, bool INTERLEAVED>
__global__ void __launch_bounds__(kInt4Threads, kRopeCtas) qk_norm_rope_kernel(const RopeArgs a) {
    griddep_wait();
    griddep_launch_dependents();
    constexpr int kLanes = D / 16;
    constexpr int kHeads = 32 / kLanes;  // heads a step
    const int lane = threadIdx.x & 31;
    const int l = lane % kLanes;
    // the warp's run of all tokens' steps, end to end
    const uint32_t unit = (blockIdx.x * kInt4Threads + threadIdx.x) >> 5;
    if (unit >= a.warps) return;
    const uint32_t s0 = unit * a.run + min(unit, a.longer);
    const uint32_t s1 = s0 + a.run + (unit < a.longer ? 1u : 0u);
    // A place in the run: a token, the kind (0: q, 1: k, 2: v) of the step's heads,
    // the steps left of that kind, and this lane's head.
    struct Place {
        uint32_t tok, b, t;
        int kind, left, h;
    };
    constexpr int kKinds = APPEND ? 3 : 2;
    auto locate = [&](Place& p, uint32_t step) {
        p.tok = a.steps.div(step);
        p.b = a.divT.div(p.tok);
        p.t = p.tok - p.b * a.divT.d;
        int i = static_cast<int>(step - p.tok * a.steps.d);
        p.kind = i < a.q_steps ? 0 : i < a.q_steps + a.kv_steps ? 1 : 2;
        if (p.kind > 0) i -= a.q_steps;
        if (p.kind > 1) i -= a.kv_steps;
        p.left = (p.kind == 0 ? a.q_steps : a.kv_steps) - i;
        p.h = i * kHeads + lane / kLanes;
    };
    // to the next step; true if its heads are not the next ones of the same kind
    auto next = [&](Place& p) {
        p.h += kHeads;
        if (--p.left > 0) return false;
        p.h = lane / kLanes;
        if (++p.kind == kKinds) {
            p.kind = 0;
            ++p.tok;
            p.b = a.divT.div(p.tok);
            p.t = p.tok - p.b * a.divT.d;
        }
        p.left = p.kind == 0 ? a.q_steps : a.kv_steps;
        return true;
    };
    Place cur;
    locate(cur, s0);

    // runs (in units of 8 elements): the pairs' halves of the rotated part, and
    // the halves of what is behind it; of v, and interleaved, halves of the row
    const int rot_lanes = a.rot / 16;
    const bool natural = INTERLEAVED || a.rot == D;
    const int pair0 = natural || l < rot_lanes ? l : rot_lanes + l;
    const int pair1 = natural ? l + kLanes : l < rot_lanes ? rot_lanes + l : kLanes + l;
    // rows come through shared memory, kRopeDepth steps ahead; a lane reads back
    // what it asked for itself
    __shared__ uint4 ring[kInt4Threads / 32][kRopeDepth][2][32];
    uint4(*mine)[2][32] = ring[threadIdx.x >> 5];
    Place ahead = cur;
    uint32_t asked = s0;
    const uint16_t *src0, *src1;  // the lane's runs of head ahead.h
    long long src_step;
    auto aim = [&]() {
        const Place& p = ahead;
        const uint16_t* x = p.kind == 0 ? a.q + p.b * a.q_sb + p.t * a.q_st
                            : p.kind == 1 ? a.k + p.b * a.k_sb + p.t * a.k_st
                                          : a.v + p.b * a.v_sb + p.t * a.v_st;
        const long long sh = p.kind == 0 ? a.q_sh : p.kind == 1 ? a.k_sh : a.v_sh;
        x += p.h * sh;
        src0 = x + 8 * (p.kind == 2 ? l : pair0);
        src1 = x + 8 * (p.kind == 2 ? l + kLanes : pair1);
        src_step = sh * kHeads;
    };
    aim();
    auto ask = [&]() {
        if (asked < s1) {
            if (ahead.h < (ahead.kind == 0 ? a.Hq : a.Hkv)) {
                uint4(*slot)[32] = mine[(asked - s0) % kRopeDepth];
                cp_async<16>(smem_addr(&slot[0][lane]), src0);
                cp_async<16>(smem_addr(&slot[1][lane]), src1);
            }
            if (++asked < s1) {
                if (next(ahead)) {
                    aim();
                } else {
                    src0 += src_step;
                    src1 += src_step;
                }
            }
        }
        cp_async_commit();
    };
#pragma unroll 1
    for (int i = 0; i < kRopeDepth; ++i) ask();

    // cos and sin of the lane's pairs: 8 of one run pair, or 4 of each run
    const bool turn0 = INTERLEAVED ? pair0 < 2 * rot_lanes : l < rot_lanes;
    const bool turn1 = INTERLEAVED ? pair1 < 2 * rot_lanes : turn0;
    float2 cs[8];
    auto load_cs = [&](uint32_t tok) {
        auto position = [&](int axis) { return a.pos[static_cast<long long>(axis) * a.tokens + tok]; };
        auto axis_of = [&](int j) { return a.axes == 1 ? 0 : (j >= a.s1) + (j >= a.s2) + (j >= a.s3); };
        // `count` pairs from j on, into cs[at ...]; a position outside the table leaves NaN in the row
        auto fetch = [&](int at, int j, auto n) {
            constexpr int kCount = decltype(n)::value;
            if (axis_of(j) == axis_of(j + kCount - 1)) {
                const int p = position(axis_of(j));
                const bool in = p >= 0 && p < a.max_pos;
                const float4* src = reinterpret_cast<const float4*>(
                    a.table + (in ? static_cast<long long>(p) * (a.rot / 2) + j : 0));
#pragma unroll
                for (int i = 0; i < kCount; i += 2) {
                    const float4 v = in ? src[i / 2] : make_float4(NAN, NAN, NAN, NAN);
                    cs[at + i] = make_float2(v.x, v.y);
                    cs[at + i + 1] = make_float2(v.z, v.w);
                }
            } else {
#pragma unroll
                for (int i = 0; i < kCount; ++i) {
                    const int p = position(axis_of(j + i));
                    cs[at + i] = p >= 0 && p < a.max_pos
                                     ? a.table[static_cast<long long>(p) * (a.rot / 2) + j + i]
                                     : make_float2(NAN, NAN);
                }
            }
        };
        if constexpr (INTERLEAVED) {
            if (turn0) fetch(0, pair0 * 4, std::integral_constant<int, 4>{});
            if (turn1) fetch(4, pair1 * 4, std::integral_constant<int, 4>{});
        } else {
            if (turn0) fetch(0, l * 8, std::integral_constant<int, 8>{});
        }
    };

    // where the outputs of cur's token and kind are: head 0's row of q_out or k_out,
    // or of the caches (-1: the cache does not have it)
    uint4* out = nullptr;
    const long long out_head = static_cast<long long>(a.T) * (D / 8);
    long long row0 = -1;
    auto enter = [&]() {
        if (!APPEND || cur.kind == 0) {
            out = reinterpret_cast<uint4*>(cur.kind == 0 ? a.q_out : a.k_out) +
                  (static_cast<long long>(cur.b) * (cur.kind == 0 ? a.Hq : a.Hkv) * a.T + cur.t) * (D / 8);
        } else {
            const long long pos = (a.starts ? static_cast<long long>(a.starts[cur.b]) : a.t0) + cur.t;
            row0 = pos >= 0 && pos < a.S_cap ? static_cast<long long>(cur.b) * a.Hkv * a.S_cap + pos : -1;
        }
    };
    enter();

    float w0[8], w1[8];
    int weights = -1;              // the kind they are of
    uint32_t cs_tok = 0xffffffffu;  // the token cs is of
    for (uint32_t s = s0; s < s1; ++s) {
        const int kind = cur.kind, h = cur.h;
        const bool store = h < (kind == 0 ? a.Hq : a.Hkv);
        cp_async_wait<kRopeDepth - 1>();
        uint4(*slot)[32] = mine[(s - s0) % kRopeDepth];
        float f0[8], f1[8];  // of heads that do not exist: whatever the slot held; nothing comes of it
        unpack8<BF16>(slot[0][lane], f0);
        unpack8<BF16>(slot[1][lane], f1);
        if (kind != 2) {
            if (cur.tok != cs_tok) load_cs(cs_tok = cur.tok);
            if (kind != weights) {
                weights = kind;
                const uint16_t* w = kind == 0 ? a.q_w : a.k_w;
#pragma unroll
                for (int j = 0; j < 8; ++j) w0[j] = w1[j] = 1.0f;
                if (w) {
                    unpack8<BF16>(reinterpret_cast<const uint4*>(w)[pair0], w0);
                    unpack8<BF16>(reinterpret_cast<const uint4*>(w)[pair1], w1);
                }
            }
            const float inv = APPEND ? inv_rms_exact<D>(f0, f1, a.eps) : inv_rms<D>(f0, f1, a.eps, store);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                f0[j] = __fmul_rn(__fmul_rn(f0[j], inv), w0[j]);
                f1[j] = __fmul_rn(__fmul_rn(f1[j], inv), w1[j]);
            }
            if constexpr (INTERLEAVED) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (turn0) rotate_pair<APPEND>(f0[2 * j], f0[2 * j + 1], cs[j], f0[2 * j], f0[2 * j + 1]);
                    if (turn1) rotate_pair<APPEND>(f1[2 * j], f1[2 * j + 1], cs[4 + j], f1[2 * j], f1[2 * j + 1]);
                }
            } else if (turn0) {
#pragma unroll
                for (int j = 0; j < 8; ++j) rotate_pair<APPEND>(f0[j], f1[j], cs[j], f0[j], f1[j]);
            }
        }
        if (!APPEND || kind == 0) {
            if (store) {
                uint4* dst = out + static_cast<long long>(h) * out_head;
                dst[pair0] = make_uint4(pack2<BF16>(f0[0], f0[1]), pack2<BF16>(f0[2], f0[3]),
                                        pack2<BF16>(f0[4], f0[5]), pack2<BF16>(f0[6], f0[7]));
                dst[pair1] = make_uint4(pack2<BF16>(f1[0], f1[1]), pack2<BF16>(f1[2], f1[3]),
                                        pack2<BF16>(f1[4], f1[5]), pack2<BF16>(f1[6], f1[7]));
            }
        } else if constexpr (APPEND) {
            if (!natural && kind == 1) {
                // runs into their natural order: run r is in lane `from`, first or second
                float n0[8], n1[8];
                const int tail = kLanes - rot_lanes;  // lanes behind the rotated part
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const int r = l + s * kLanes;
                    const bool is_second = r < 2 * rot_lanes ? r >= rot_lanes : r - 2 * rot_lanes >= tail;
                    const int from = lane - l + (r < 2 * rot_lanes ? (is_second ? r - rot_lanes : r)
                                                                   : r - rot_lanes - (is_second ? tail : 0));
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float p = __shfl_sync(0xffffffffu, f0[j], from);
                        const float q = __shfl_sync(0xffffffffu, f1[j], from);
                        (s == 0 ? n0 : n1)[j] = is_second ? q : p;
                    }
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) f0[j] = n0[j], f1[j] = n1[j];
            }
            const bool ok = store && row0 >= 0;
            const long long row = row0 + static_cast<long long>(h) * a.S_cap;
            store_int4_runs<D, BS>(f0, f1, l, row, ok, kind == 1 ? a.kc : a.vc, kind == 1 ? a.kp : a.vp);
        }
        if (s + 1 < s1 && next(cur)) enter();
        ask();  // into the slot that has been used
    }
}

}  // namespace tqkv
