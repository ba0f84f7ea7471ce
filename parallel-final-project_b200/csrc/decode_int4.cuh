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
//   score_t = sum_blocks (scale_t u) (codes . q) + zero_t (sum of u q over the block)
//   O       = [ sum_t (p_t scale_t) codes_t + sum_t p_t zero_t ] / sum_t p_t
// with u = log2(e) / sqrt(D): a score is then a power of two times its logarithm
// of two.  The block scale is applied to the score in fp32; for V it is multiplied into
// p in fp32 before p is rounded to fp16 as the product's operand (relative
// error 2^-11 a token, like the 16-bit P of any tensor-core attention; Copies and
// Rests, below, take it out of fp16 outputs).  The zero sums stay in fp32.
//
// V's codes enter as code - 8 for even tokens and code - 7 for odd ones (one
// packed fp16 subtraction, exact) beside zero + 8 scale and zero + 7 scale:
// sums of codes 0..15 would grow with the length while O does not, and what
// the tensor core cuts off each sum, and p's rounding, would grow with them.
// K's zero terms are a product as well: a column of zeros times the blocks'
// sums of q in two fp16 words, 2^14 above the codes' unit, so that they hold all
// that fp32 does: keys with a large mean have zeros far above their scales (with
// the words in the codes' unit, off by 2^-15 of the largest |q|, zeros of 4000 moved O
// by 1 to 4 %).  B1 H32 S65536 52.3 -> 52.5 us.
//
// Range.  p * scale must stay inside fp16 whatever the caches hold: the
// operand is 2^(score - M - e + 11) * scale with M within 2^4 of the largest
// score so far and 2^e above the largest scale, so it is below 2^15, and
// tokens 2^-24 of the largest keep all their bits.  fp32 holds M + e - 11 to 1 / 4 up
// to 2^22.  Scores that fp16's q and K reach (2^38) leave no place for e there, and
// the weights would leave the operand's range by a rounding of the reference (q = K =
// 1000 gave NaN); beyond 2^22 the reference is therefore M itself, the largest score,
// whose weight is 1 then: exactly, as the score's unit is a power of two.
//
// Copies.  Over many tokens O is a sum of terms that cancel, and the operands'
// rounding shows beside fp16's own: 3.2e-4 of O in the mean, where an O rounded
// once is 2.0e-4 off (S = 131,072).  Of the 8 columns of the products a group of
// up to 4 heads leaves half or more idle; for fp16 they hold copies of the heads
// whose references are 1 / 2, 1 / 4 or 1 / 8 of an octave apart, so that every copy
// rounds other numbers, and O is their mean: 2.2e-4 with 8 copies.  The stream
// takes as long as before; the mean costs a piece 0.3 to 0.8 us (B1 H32 S65536
// 51.9 -> 52.3 us, 512 heads of one row 4.3 -> 4.9 us).  Remainders of the weights
// in the idle columns gave 2.0e-4, but 55.3 us.  bf16's rounding covers all of it.
//
// Rests.  fp16 groups of 5 and more have no column to spare, and O was 1.5 to 1.6 times as
// far off as one rounded once.  What rounding takes off the operand is a second
// operand there, rounded to fp16 itself (2^-22): 3.2e-4 -> 2.1e-4, which is O's own
// rounding.  32 ragged sequences, 64/8 heads of 128: 26.6 -> 27.3 us (block 128), 28.7 ->
// 31.8 (block 32); 64/4 heads 26.4 -> 29.8; B4 64/8 heads S65536 54 -> 65.
//
// Work split.  Units are (sequence, KV head, slice of 8 * NT query heads); a
// unit has ceil(length / 16) granules, and counts for six more, about what
// starting and ending it costs (ragged lengths put many short units into one
// run: 37.3 us without, 30.9 with it for 32 sequences of 1 to 4099 rows and 8 KV
// heads; 3, 6 and 12 are 28.3, 27.6 and 28.5 there, 23.8, 21.9 and 21.9 with heads of
// 64, 29.6, 26.6 and 26.8 with 16 query heads a KV head).  All units' granules, end to end, are cut
// into equal runs, one per CTA, and each CTA's run into equal runs, one per
// warp, whatever the lengths are.  A warp meets at most one unit that began
// before its run and one that goes on behind it; units that lie within its run
// it finishes alone, without meeting another warp.  The states (acc[D], l, its
// reference, per query head) of cut units are joined in order: within the CTA
// in shared memory at the end of the run, across CTAs through records in the
// workspace, by the CTA that arrives last at the unit's counter.  The order
// does not depend on which one that is.  The merging CTA zeroes the records
// and the counter again.
//
// Every warp streams for itself: a ring of two tiles filled by cp.async (16
// bytes a lane, past L1), waited for by group, with no barrier between warps.
// Rows behind the sequence's end are filled with zeros and are not read.
// 16-byte chunks are exchanged within a row so that both ways the tile is read
// (a row's chunks side by side for K, one chunk of every second row for V) are
// free of bank conflicts.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "device_common.cuh"
#include "kv_int4.cuh"

namespace tqkv {

constexpr int kGranule = 16;     // rows by which runs are cut
constexpr int kUnitCost = 6;     // granules that a unit counts for besides its own
constexpr int kI4MinWarps = 8;   // fewest warps of a CTA
constexpr int kCutTiles = 2;     // tiles a warp does in the time that joining a cut unit takes

// CTAs that `n` granules of `units` units are dealt to, `most` at most: enough that each warp has
// a tile (`per` granules a CTA), or as many as give each CTA whole units where all are as long,
// if a warp then has less than kCutTiles tiles more.  us without the second choice and with it:
// 16 x 8 KV heads of 300 rows (D = 128, blocks of 32) 9.9 / 6.6, 64 x 8 of 500 17.0 / 13.6 and of
// 1 10.4 / 4.3, 8 x 12 of 1024 (D = 64) 9.6 / 7.4; 19 x 8 of 1200, where the tiles decide, 13.9 / 13.9.
template <class I>
__host__ __device__ inline I int4_ctas(I n, I units, I most, I per) {
    I ctas = n / per;
    ctas = ctas > most ? most : ctas < 1 ? 1 : ctas;
    I whole = units;
    if (units > most) {
        const I each = (units + most - 1) / most;
        whole = (units + each - 1) / each;
    }
    return whole >= ctas || static_cast<long long>(n) * (ctas - whole) <
                                static_cast<long long>(kCutTiles) * per * whole * ctas
               ? whole
               : ctas;
}

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
    int stride;                 // columns of the products from a head to its next copy: 1, 2, 4; 8 without
    float score_scale;          // u = log2(e) / sqrt(D)
};

// A unit that a warp's run cuts: its first granule (-1: none, -2: the warp has
// no run), the one behind its last, its first output row b * Hq + h, and its
// query heads.
struct alignas(16) CutUnit {
    int start, end, row, nq;
};

// REST: weights as two fp16 operands, for fp16 outputs of groups without idle columns
template <int D, int BS, int NT, bool REST>
struct I4Cfg {
    static constexpr int kRow = D / 2;            // bytes of codes a row
    static constexpr int kSub = D / 32;           // 32-element groups = words per lane chunk
    static constexpr int kNS = D / BS;            // blocks a row
    static constexpr int kTile = 4096 / D;        // rows a tile: 2 KB of codes
    static constexpr int kM = kTile / 16;         // granules a tile
    static constexpr int kQ = 8 * NT;             // query heads a unit takes
    static constexpr int kKV = kTile * kRow;
    static constexpr int kSc = kTile * kNS * 4;
    static constexpr int kStage = 2 * (kKV + kSc);
    // A tile in use and one on its way.  A third stage gains 1 to 4 % where blocks of
    // 64 and more leave the kernel waiting for memory, and costs 6 % with blocks of 32.
    static constexpr int kStages = 2;
    static constexpr int kRecStride = D + 4;      // acc[D], l at D, R at D + 1
    // Warps of a CTA, one CTA an SM: 12 leave each 168 registers, 8 leave 255.  12
    // hide more latency (B1 H32 S65536, block 128: 51.9 us, 57.2 with 8 and with 16)
    // unless two sets of accumulators (NT = 2) or four blocks a row spill (B1 32/8
    // heads S65536, block 32: 25.8 us with 12, 24.0 with 8), or the weights' rests need
    // the registers (32 ragged sequences, 64/8 heads of 128, block 64: 33.0 and 29.3; of 64: 22.4
    // and 23.2).
    static constexpr int kWarps = NT == 2 || kNS == 4 || (REST && D == 128) ? 8 : 12;
    static_assert(kWarps >= kI4MinWarps, "the workspace holds a record pair for every CTA");
    // bytes of the states of `rows` query heads
    __host__ __device__ static constexpr int state(int rows) { return rows * kRecStride * 4; }
    // a warp's ring: it takes the state of the unit that goes on behind its run
    // once all its tiles are used
    __host__ __device__ static constexpr int ring(int rows) {
        return kStages * kStage > state(rows) ? kStages * kStage : state(rows);
    }
    // rings, the states of the units that began before a run, two descriptors a
    // warp, flags
    static constexpr int smem_bytes(int rows) {
        return kWarps * (ring(rows) + state(rows) + 2 * static_cast<int>(sizeof(CutUnit))) + 16;
    }
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The codes in the low (U = 24) or next (20) nibbles, less 8 in the low half (an
// even token's) and 7 in the high one, times 2^-U.
template <int U>
__device__ __forceinline__ uint32_t centred(uint32_t x) {
    const uint32_t code = x & (U == 24 ? 0x000f000fu : 0x00f000f0u);
    const uint32_t mid = U == 24 ? 0x00070008u : 0x00700080u;
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&code), *reinterpret_cast<const __half2*>(&mid));
    return *reinterpret_cast<const uint32_t*>(&v);
}

// transpose of an 8 x 8 matrix of 16-bit values held two to a lane
__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}

// Four 8 x 8 matrices of 16-bit values from shared memory, transposed: lane i
// gives the address of row i % 8 of matrix i / 8.
__device__ __forceinline__ void ldmatrix_trans(uint32_t (&r)[4], const uint8_t* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_addr(p))
                 : "memory");
}

// N words from shared memory by one load
template <int N>
__device__ __forceinline__ void lds_words(uint32_t (&w)[N], const uint8_t* p) {
    if constexpr (N == 4) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p);
    else if constexpr (N == 2) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
    else w[0] = *reinterpret_cast<const uint32_t*>(p);
}

__device__ __forceinline__ int i4_length(const Int4DecodeArgs& a, int b) {
    if (a.lengths == nullptr) return a.S;
    const int n = a.lengths[b];
    return n < 0 ? 0 : n > a.S ? a.S : n;
}

// Arrives at a counter: everything that this CTA wrote before the barrier in
// front of it is visible to whoever sees the counter's new value.
__device__ __forceinline__ unsigned int arrive_acq_rel(unsigned int* p) {
    unsigned int before;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(p) : "memory");
    return before;
}

// Four elements of an output row.
__device__ __forceinline__ void store_out(uint16_t* dst, float4 v, int bf16) {
    uint2 out;
    out.x = bf16 ? pack2<true>(v.x, v.y) : pack2<false>(v.x, v.y);
    out.y = bf16 ? pack2<true>(v.z, v.w) : pack2<false>(v.z, v.w);
    *reinterpret_cast<uint2*>(dst) = out;
}

// (v, lr) += (x, xr): sums and their l relative to 2^reference; empty states
// have l = 0 at -infinity.
__device__ __forceinline__ void join(float4& v, float2& lr, float4 x, float2 xr) {
    const float m = fmaxf(lr.y, xr.y);
    const float f = lr.y == m ? 1.0f : fast_exp2(lr.y - m);
    const float e = xr.y == m ? 1.0f : fast_exp2(xr.y - m);
    v.x = fmaf(x.x, e, v.x * f);
    v.y = fmaf(x.y, e, v.y * f);
    v.z = fmaf(x.z, e, v.z * f);
    v.w = fmaf(x.w, e, v.w * f);
    lr = make_float2(fmaf(xr.x, e, lr.x * f), m);
}

// Granules that a unit of `len` rows counts for.
__device__ __forceinline__ int unit_length(int len) {
    return len > 0 ? (len - 1) / kGranule + 1 + kUnitCost : 0;
}

// The unit that a place in the granules' sequence belongs to, moved forward.
struct UnitWalk {
    int b, kvh, slice;  // sequence; KV head and slice of its query heads
    int len, nt;  // its rows, and what it counts for
    int start;    // its first place; its first granule is kUnitCost behind

    __device__ __forceinline__ int first() const { return start + kUnitCost; }
    __device__ __forceinline__ int end() const { return start + nt; }

    __device__ __forceinline__ void load(const Int4DecodeArgs& a) {
        len = b < a.B ? i4_length(a, b) : 0;
        nt = unit_length(len);
    }
    // g below the total: the loop ends
    __device__ __forceinline__ void seek(const Int4DecodeArgs& a, int g) {
        while (g >= start + nt && b < a.B) {
            start += nt;
            if (nt > 0) {
                if (++slice < a.slices) continue;
                slice = 0;
                if (++kvh < a.Hkv) continue;
            }
            kvh = 0;
            ++b;
            load(a);
        }
    }
};

static_assert(I4Cfg<128, 32, 1, false>::smem_bytes(8) <= 227 * 1024 &&
                  I4Cfg<128, 32, 2, false>::smem_bytes(16) <= 227 * 1024,
              "the stages and the states of any group fit");

template <int D, int BS, int NT, bool REST>
__global__ void __launch_bounds__(I4Cfg<D, BS, NT, REST>::kWarps * 32, 1)
    decode_int4_kernel(const Int4DecodeArgs a, int bf16) {
    using C = I4Cfg<D, BS, NT, REST>;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int nw = C::kWarps;
    const int g = lane >> 2, c = lane & 3;  // the mma's row and column groups
    const int rows = a.rec_rows;
    const int ring_bytes = C::ring(rows);
    const int state_floats = rows * C::kRecStride;
    uint8_t* ring = smem + warp * ring_bytes;
    float* merge = reinterpret_cast<float*>(smem + nw * ring_bytes);  // [warp] state
    CutUnit* cuts = reinterpret_cast<CutUnit*>(merge + nw * state_floats);  // [warp][2]
    unsigned int* flags = reinterpret_cast<unsigned int*>(cuts + 2 * nw);   // [2]
    griddep_wait();
    griddep_launch_dependents();

    // ---- this CTA's granules [g0, g1) of all units' n: n / ctas each, one more for
    // the first n % ctas CTAs
    const int per_seq = a.Hkv * a.slices;
    int n = 0, of_lane = 0;  // of sequence `lane`
    int units = 0;           // sequences that hold something
    bool empty = false;
    if (a.lengths == nullptr) {
        n = a.B * unit_length(a.S);
        empty = a.S == 0;
    } else {
        for (int b = lane; b < a.B; b += 32) {
            const int len = i4_length(a, b);
            const int x = unit_length(len);
            if (b == lane) of_lane = x;
            n += x;
            empty |= len == 0;
            units += len != 0;
        }
#pragma unroll
        for (int off = 16; off; off >>= 1) n += __shfl_xor_sync(0xffffffffu, n, off);
        units = __reduce_add_sync(0xffffffffu, units);
        empty = __any_sync(0xffffffffu, empty);
    }
    n *= per_seq;
    if (empty) {  // heads of sequences that hold nothing come out as zero
        for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
            if (i4_length(a, b) != 0) continue;
            uint32_t* o = reinterpret_cast<uint32_t*>(a.o) + static_cast<long long>(b) * a.Hq * (D / 2);
            for (int i = threadIdx.x; i < a.Hq * (D / 2); i += blockDim.x) o[i] = 0u;
        }
    }
    const unsigned ctas = a.lengths == nullptr ? gridDim.x
                                               : int4_ctas<unsigned>(n, units * per_seq, gridDim.x, nw * C::kM);
    const unsigned cta = blockIdx.x;
    if (cta >= ctas || n == 0) return;
    const unsigned each = n / ctas, more = n - each * ctas;
    const int g0 = cta * each + (cta < more ? cta : more);
    const int g1 = g0 + each + (cta < more ? 1 : 0);
    auto cta_of = [&](unsigned tile) {
        const unsigned edge = more * (each + 1);
        return tile < edge ? tile / static_cast<unsigned>(each + 1) : more + static_cast<unsigned>(tile - edge) / each;
    };
    // rounded up: warp 0 has a granule, so that a unit that began before this CTA is its first
    const int w0 = g0 + ((g1 - g0) * warp + nw - 1) / nw, w1 = g0 + ((g1 - g0) * (warp + 1) + nw - 1) / nw;

    UnitWalk walk;  // of the unit being worked on
    walk.start = 0;
    walk.b = 0;
    walk.kvh = walk.slice = 0;
    walk.len = walk.nt = 0;
    if (w0 < w1) {
        if (a.lengths == nullptr) {
            const unsigned each_b = per_seq * unit_length(a.S);
            walk.b = static_cast<unsigned>(w0) / static_cast<unsigned>(each_b);
            walk.start = walk.b * each_b;
        } else {
            for (int base = 0; base < a.B; base += 32) {
                const int b = base + lane;
                int x = base == 0 ? of_lane
                        : b < a.B ? unit_length(i4_length(a, b))
                                  : 0;
                x *= per_seq;
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, x, off);
                    if (lane >= off) x += y;
                }
                // sequences of these 32 that end at or before w0
                const int k = __popc(__ballot_sync(0xffffffffu, walk.start + x <= w0));
                if (k > 0) {
                    walk.start += __shfl_sync(0xffffffffu, x, k - 1);
                    walk.b = base + k;
                }
                if (k < 32) break;
            }
        }
        walk.load(a);
        const unsigned u = static_cast<unsigned>(w0 - walk.start) / static_cast<unsigned>(walk.nt);
        walk.kvh = a.slices == 1 ? u : u / static_cast<unsigned>(a.slices);
        walk.slice = u - walk.kvh * a.slices;
        walk.start += u * walk.nt;
    }
    if (lane < 2) cuts[2 * warp + lane].start = w0 < w1 ? -1 : -2;
    __syncwarp();

    // ---- the warp's stream of tiles, each of up to kM granules of one unit
    constexpr int kChunks = C::kRow / 16;          // 16-byte chunks a row
    constexpr int kRowsPerCopy = 32 / kChunks;     // rows one cp.async of the warp covers
    const int copy_row = lane / kChunks;
    // chunk i of row t stands at i ^ (t / 2 % 4), or i ^ (t / 4 % 2) for D = 64
    const int copy_pos = (lane % kChunks) ^ (C::kSub == 4 ? (copy_row >> 1) & 3 : (copy_row >> 2) & 1);
    const uint32_t copy_dst = smem_addr(ring) + copy_row * C::kRow + copy_pos * 16;
    const uint32_t par_dst = smem_addr(ring) + 2 * C::kKV + lane * 4 * C::kNS;
    UnitWalk ahead = walk;
    int next = w0, ahead_left = 0;      // granule behind the unit's part; its rows not yet asked for
    const uint8_t* k_src = nullptr;     // where the next tile's rows are, this lane's part
    const uint32_t* kp_src = nullptr;
    const long long k_to_v = a.vq - a.kq, kp_to_vp = a.vs - a.ks;
    uint32_t fill = 0;                  // offset of the stage to fill next
    auto issue = [&]() {
        while (ahead_left <= 0 && next < w1) {
            ahead.seek(a, next);
            const int from = next > ahead.first() ? next : ahead.first();
            next = ahead.end() < w1 ? ahead.end() : w1;
            if (from >= next) continue;
            const int t0 = (from - ahead.first()) * kGranule;
            const int rows = (next - ahead.first()) * kGranule;
            ahead_left = (rows < ahead.len ? rows : ahead.len) - t0;
            const long long row =
                (static_cast<long long>(ahead.b) * a.Hkv + ahead.kvh) * a.S_cap + t0;
            k_src = a.kq + row * C::kRow + lane * 16;
            kp_src = a.ks + (row + lane) * C::kNS;
        }
        if (ahead_left > 0) {
            const uint8_t* v_src = k_src + k_to_v;
            const uint32_t* vp_src = kp_src + kp_to_vp;
            const uint32_t dst = copy_dst + fill, pdst = par_dst + fill;
            if (ahead_left >= C::kTile) {
#pragma unroll
                for (int i = 0; i < C::kKV / 512; ++i) {
                    cp_async<16>(dst + i * 512, k_src + i * 512);
                    cp_async<16>(dst + C::kKV + i * 512, v_src + i * 512);
                }
#pragma unroll
                for (int i = 0; i < C::kTile / 32; ++i) {
                    cp_async<4 * C::kNS>(pdst + i * 128 * C::kNS, kp_src + i * 32 * C::kNS);
                    cp_async<4 * C::kNS>(pdst + C::kSc + i * 128 * C::kNS, vp_src + i * 32 * C::kNS);
                }
            } else {
                // rows that are not the run's: zeros, addressed at the tile's first row
#pragma unroll 1
                for (int i = 0; i < C::kKV / 512; ++i) {
                    const bool real = copy_row + i * kRowsPerCopy < ahead_left;
                    const int o = real ? i * 512 : -copy_row * C::kRow;
                    cp_async<16>(dst + i * 512, k_src + o, real);
                    cp_async<16>(dst + C::kKV + i * 512, v_src + o, real);
                }
#pragma unroll
                for (int i = 0; i < C::kTile / 32; ++i) {
                    const bool real = lane + i * 32 < ahead_left;
                    const int o = (real ? i * 32 : -lane) * C::kNS;
                    cp_async<4 * C::kNS>(pdst + i * 128 * C::kNS, kp_src + o, real);
                    cp_async<4 * C::kNS>(pdst + C::kSc + i * 128 * C::kNS, vp_src + o, real);
                }
            }
            ahead_left -= C::kTile;
            k_src += C::kKV;
            kp_src += C::kTile * C::kNS;
            fill = C::kStage - fill;
        }
        cp_async_commit();  // a group for every tile, real or not, so that groups can be counted
    };
    // ---- the query heads of a unit, as they are in memory: lane (g, c) takes 8
    // elements of every 32 of head g; asked for ahead of the tiles
    uint4 q_raw[NT][C::kSub];
    auto load_q = [&](const UnitWalk& unit) {
        const int left = a.group - unit.slice * C::kQ;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int head = t * 8 + (NT == 1 ? g & (a.stride - 1) : g);
            const bool has = head < left;
            const uint4* src = reinterpret_cast<const uint4*>(
                a.q + (static_cast<long long>(unit.b) * a.Hq + unit.kvh * a.group + unit.slice * C::kQ +
                       (has ? head : 0)) * D);
#pragma unroll
            for (int b = 0; b < C::kSub; ++b)
                q_raw[t][b] = has ? src[b * 4 + c] : make_uint4(0, 0, 0, 0);
        }
    };
    if (w0 < w1) load_q(walk);
#pragma unroll 1
    for (int i = 0; i < C::kStages; ++i) issue();

    const float middle = g & 1 ? 7.0f : 8.0f;  // what centred() takes off tokens g and g + 8
    const uint8_t* buf = ring;
    // this lane's place in a tile: row g's and row 2c's chunks
    const int k_at = g * C::kRow + (C::kSub == 4 ? (c ^ ((g >> 1) & 3)) * 16
                                                 : (((c >> 1) ^ ((g >> 2) & 1)) * 16 + (c & 1) * 8));
    const int mr = lane & 7, mi = lane >> 3;  // row and matrix that it addresses
    const int v_at =
        BS == 128  ? mr * C::kRow + (mi ^ ((mr >> 1) & 3)) * 16
        : BS == D  ? (mr + (mi >> 1) * 8) * C::kRow + ((mi & 1) ^ ((mr >> 2) & 1)) * 16
        : C::kSub == 4 ? 2 * c * C::kRow + ((g >> 1) ^ c) * 16
                       : 2 * c * C::kRow + ((g >> 2) ^ (c >> 1)) * 16 + ((g >> 1) & 1) * 8;
    // first element of the four that row g of fragment pair b stands for
    auto element = [&](int b) {
        return BS == 128 ? 32 * (g >> 1) + 8 * b + 4 * (g & 1)
               : BS == D ? 32 * ((g >> 1) & 1) + 8 * (2 * b + (g >> 2)) + 4 * (g & 1)
                         : 32 * b + 4 * g;
    };

    for (int mine = w0; mine < w1;) {
        // ---- one piece: the warp's granules [mine, p1) of one unit
        const UnitWalk cur = walk;
        const int from = mine > cur.first() ? mine : cur.first();
        const int p1 = cur.end() < w1 ? cur.end() : w1;
        mine = p1;
        if (from >= p1) {  // the run ends before the unit's first granule
            if (mine < w1) {
                walk.seek(a, mine);
                load_q(walk);
            }
            continue;
        }
        const bool began_before = from != cur.first();
        const bool whole = !began_before && p1 == cur.end();
        const int head0 = cur.kvh * a.group + cur.slice * C::kQ;
        const int left_heads = a.group - cur.slice * C::kQ;
        const int nq = left_heads < C::kQ ? left_heads : C::kQ;

        // ---- q of the unit as the products' right operands
        // u, and from the codes' 2^-24 to the sums' 2^-10: a factor of the blocks' scales, or of the
        // score, its zero terms lowered first, where that is fewer products (32 ragged sequences,
        // blocks of 32: 28.4 us by the first way, 27.9 by the second)
        constexpr bool kScaleBlocks = C::kNS <= 2 * NT;
        const float unit = 16384.0f * a.score_scale;
        uint32_t qf[NT][C::kSub][2][2], qz[NT];
        float sc[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float f[C::kSub][8];
            float amax = 0.0f;
#pragma unroll
            for (int b = 0; b < C::kSub; ++b) {
                if (bf16) unpack8<true>(q_raw[t][b], f[b]);
                else unpack8<false>(q_raw[t][b], f[b]);
#pragma unroll
                for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(f[b][i]));
            }
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            // 2^e with max |q| * 2^e in [2^14, 2^15): exact in fp16, also over 16, down
            // to 2^-24 of the largest element; an infinite one stays so
            int e = 141 - static_cast<int>(__float_as_uint(amax) >> 23);
            e = amax == 0.0f ? 0 : e > 100 ? 100 : e;
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
            // block c's sum (below 2^22) * 2^-10 (and u) as a sum of two fp16, against its zero twice:
            // off by 2^-23 of it or 2^-25, which is 2^-26 of the largest |q| at most
            float mine_sum = 0.0f;
#pragma unroll
            for (int s = 0; s < C::kNS; ++s) {
                sum[s] += __shfl_xor_sync(0xffffffffu, sum[s], 1);
                sum[s] += __shfl_xor_sync(0xffffffffu, sum[s], 2);
                if (c == s) mine_sum = sum[s] * 0.0009765625f * (kScaleBlocks ? a.score_scale : 1.0f);
            }
            const float high = __half2float(__float2half_rn(mine_sum));
            qz[t] = pack2<false>(high, mine_sum - high);
            // the scores' columns in this lane are heads 2c and 2c + 1.  2^(10 - e), or 2^80: sums
            // differ by 2^-60 if at all (codes * 2^-24, q and scales of 2^-24 each, the unit's 2^12 and
            // more), so that all but the largest then weigh nothing either way, and are below 2^34:
            // no score overflows
            const float down = fminf(__uint_as_float(static_cast<uint32_t>(127 - e) << 23) * 1024.0f, 0x1p80f);
            sc[t][0] = __shfl_sync(0xffffffffu, down, 8 * c);
            sc[t][1] = __shfl_sync(0xffffffffu, down, 8 * c + 4);
        }

        // R = M + e - 11, M the largest score (base 2) so far, or up to 4 less, and `limit` the
        // raw score beyond which R has to move, M + 4; far from 0 R = M, the largest, and `limit` too
        constexpr float kFar = 4194304.0f;
        float acc[NT][C::kSub][2][4], zsum[NT][C::kNS][2], R[NT][2], limit[NT][2], l[NT][2];
        float scale_top = 0.0f;  // 2^e
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int b = 0; b < C::kSub; ++b)
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[t][b][i >> 2][i & 3] = 0.0f;
#pragma unroll
            for (int s = 0; s < C::kNS; ++s) zsum[t][s][0] = zsum[t][s][1] = 0.0f;
            R[t][0] = R[t][1] = limit[t][0] = limit[t][1] = -INFINITY;
            l[t][0] = l[t][1] = 0.0f;
        }

        // ---- the piece's tiles
        const int run_rows = (p1 - cur.first()) * kGranule;
        const int piece_rows = run_rows < cur.len ? run_rows : cur.len;
        for (int left = piece_rows - (from - cur.first()) * kGranule; left > 0; left -= C::kTile) {
            cp_async_wait<C::kStages - 1>();
            __syncwarp();
            const uint8_t* kp = buf + 2 * C::kKV + g * 4 * C::kNS;
            const uint8_t* vp = kp + C::kSc;

            // scores of the tile, in units where 2^(s * sc) is the weight
            float s[NT][C::kM][4];
#pragma unroll
            for (int m = 0; m < C::kM; ++m) {
                uint32_t w0[C::kSub], w1[C::kSub], q0[C::kNS], q1[C::kNS];
                lds_words(w0, buf + k_at + m * 16 * C::kRow);
                lds_words(w1, buf + k_at + (m * 16 + 8) * C::kRow);
                lds_words(q0, kp + m * 16 * 4 * C::kNS);
                lds_words(q1, kp + (m * 16 + 8) * 4 * C::kNS);
                // zero terms: block c's zero twice, against the two words of its sum of q
                uint32_t z0 = q0[0], z1 = q1[0];
                if constexpr (C::kNS > 1) {
                    z0 = *reinterpret_cast<const uint32_t*>(kp + (m * 16 * C::kNS + c % C::kNS) * 4);
                    z1 = *reinterpret_cast<const uint32_t*>(kp + ((m * 16 + 8) * C::kNS + c % C::kNS) * 4);
                }
                z0 = __byte_perm(z0, z0, 0x3232);
                z1 = __byte_perm(z1, z1, 0x3232);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[t][m][i] = 0.0f;
                    mma_f16(s[t][m], z0, z1, 0u, 0u, qz[t], 0u);
                }
                if constexpr (!kScaleBlocks) {
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[t][m][i] *= 6.103515625e-05f;
                }
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
                        float a0 = __low2float(*reinterpret_cast<const __half2*>(&q0[blk]));
                        float a1 = __low2float(*reinterpret_cast<const __half2*>(&q1[blk]));
                        if constexpr (kScaleBlocks) a0 *= unit, a1 *= unit;
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                s[t][m][i] = fmaf(d[t][i], i < 2 ? a0 : a1, s[t][m][i]);
                    }
                }
                if constexpr (!kScaleBlocks) {
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[t][m][i] *= unit;
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

            // ---- do the references still hold?
            __half2 big = __half2half2(__ushort_as_half(0));
#pragma unroll
            for (int m = 0; m < C::kM; ++m)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    uint32_t vpar[C::kNS];
                    lds_words(vpar, vp + (m * 16 + 8 * r) * 4 * C::kNS);
#pragma unroll
                    for (int k = 0; k < C::kNS; ++k)
                        big = __hmax2(big, *reinterpret_cast<const __half2*>(&vpar[k]));
                }
            bool over = __low2float(big) > scale_top;
            float top[NT][2];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    top[t][j] = fmaxf(s[t][0][j], s[t][0][j + 2]);
#pragma unroll
                    for (int m = 1; m < C::kM; ++m)
                        top[t][j] = fmaxf(top[t][j], fmaxf(s[t][m][j], s[t][m][j + 2]));
                    over |= top[t][j] > limit[t][j];
                }
            if (__any_sync(0xffffffffu, over)) {
                float bigf = fmaxf(__low2float(big), 5.9604644775390625e-08f);
#pragma unroll
                for (int off = 4; off < 32; off <<= 1)
                    bigf = fmaxf(bigf, __shfl_xor_sync(0xffffffffu, bigf, off));
                // the power of two above, and its exponent
                scale_top = fmaxf(scale_top,
                                  __uint_as_float((__float_as_uint(bigf) + 0x00800000u) & 0x7f800000u));
                const float e = static_cast<float>(static_cast<int>(__float_as_uint(scale_top) >> 23) - 127);
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float x = top[t][j] * sc[t][j];
#pragma unroll
                        for (int off = 4; off < 32; off <<= 1)
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
                        // copy i of a head: i / copies higher
                        const float up = NT == 1 ? 0.125f * static_cast<float>((2 * c + j) & -a.stride) : 0.0f;
                        const float y = limit[t][j] * sc[t][j];
                        const float m = fmaxf(x, fabsf(y) > kFar ? y : y - 4.0f);
                        const float r = fabsf(m) > kFar ? m : m + (e - 11.0f + up);
                        limit[t][j] = (fabsf(m) > kFar ? m : m + 4.0f) / sc[t][j];
                        const float f = r == R[t][j] ? 1.0f : fast_exp2(R[t][j] - r);
                        R[t][j] = r;
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
                uint32_t q0[C::kNS], q1[C::kNS];  // parameters of rows g, g + 8
                lds_words(q0, vp + m * 16 * 4 * C::kNS);
                lds_words(q1, vp + (m * 16 + 8) * 4 * C::kNS);
                // 16 bits of tokens 2c, 2c + 1 (vlo) and 2c + 8, 2c + 9 (vhi): row g of the
                // V fragments.  With one block a row any 16 bits will do, and a transposing
                // load gives chunk b's; else row g's of the 32-element group b, so that a
                // fragment has one scale
                uint32_t vlo[C::kSub], vhi[C::kSub];
                const uint8_t* vt = buf + C::kKV + v_at + m * 16 * C::kRow;
                if constexpr (BS == 128) {
                    ldmatrix_trans(vlo, vt);
                    ldmatrix_trans(vhi, vt + 8 * C::kRow);
                } else if constexpr (BS == D) {
                    uint32_t r[4];
                    ldmatrix_trans(r, vt);
                    vlo[0] = r[0], vlo[1] = r[1], vhi[0] = r[2], vhi[1] = r[3];
                } else {
                    uint32_t x[4][C::kSub];
#pragma unroll
                    for (int i = 0; i < 4; ++i) lds_words(x[i], vt + ((i & 1) + (i >> 1) * 8) * C::kRow);
                    const uint32_t sel = (g & 1) ? 0x7632u : 0x5410u;
#pragma unroll
                    for (int b = 0; b < C::kSub; ++b) {
                        vlo[b] = __byte_perm(x[0][b], x[1][b], sel);
                        vhi[b] = __byte_perm(x[2][b], x[3][b], sel);
                    }
                }
                float p[NT][4];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        p[t][i] = fast_exp2(fmaf(s[t][m][i], sc[t][i & 1], -R[t][i & 1]));
                    l[t][0] += p[t][0] + p[t][2];
                    l[t][1] += p[t][1] + p[t][3];
                }
#pragma unroll
                for (int k = 0; k < C::kNS; ++k) {
                    float2 va = __half22float2(*reinterpret_cast<const __half2*>(&q0[k]));
                    float2 vb = __half22float2(*reinterpret_cast<const __half2*>(&q1[k]));
                    va.y = fmaf(va.x, middle, va.y);
                    vb.y = fmaf(vb.x, middle, vb.y);
                    uint32_t bw[NT][2], rest[NT][2];  // p * scale, and what its rounding took off
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const float scale = r == 0 ? va.x : vb.x;
                            const float w0 = p[t][2 * r] * scale, w1 = p[t][2 * r + 1] * scale;
                            const uint32_t w = pack2<false>(w0, w1);
                            bw[t][r] = movmatrix(w);
                            if constexpr (REST) {
                                const float2 have = __half22float2(*reinterpret_cast<const __half2*>(&w));
                                rest[t][r] = movmatrix(pack2<false>(w0 - have.x, w1 - have.y));
                            }
                        }
                        zsum[t][k][0] = fmaf(p[t][0], va.y, fmaf(p[t][2], vb.y, zsum[t][k][0]));
                        zsum[t][k][1] = fmaf(p[t][1], va.y, fmaf(p[t][3], vb.y, zsum[t][k][1]));
                    }
#pragma unroll
                    for (int b = k * BS / 32; b < (k + 1) * BS / 32; ++b) {
                        const uint32_t lo = vlo[b], hi = vhi[b];
                        const uint32_t lo8 = lo >> 8, hi8 = hi >> 8;
                        const uint32_t a0 = centred<24>(lo), a1 = centred<24>(lo8);
                        const uint32_t a2 = centred<24>(hi), a3 = centred<24>(hi8);
                        const uint32_t c0 = centred<20>(lo), c1 = centred<20>(lo8);
                        const uint32_t c2 = centred<20>(hi), c3 = centred<20>(hi8);
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            mma_f16(acc[t][b][0], a0, a1, a2, a3, bw[t][0], bw[t][1]);
                            mma_f16(acc[t][b][1], c0, c1, c2, c3, bw[t][0], bw[t][1]);
                            if constexpr (REST) {
                                mma_f16(acc[t][b][0], a0, a1, a2, a3, rest[t][0], rest[t][1]);
                                mma_f16(acc[t][b][1], c0, c1, c2, c3, rest[t][0], rest[t][1]);
                            }
                        }
                    }
                }
            }
            buf = buf == ring ? ring + C::kStage : ring;
            __syncwarp();  // every lane is done with the stage: refill it
            issue();
        }

        if (mine < w1) {
            walk.seek(a, mine);
            load_q(walk);
        }

        // ---- the mean of a head's copies, at the first one's reference
        if (NT == 1 && !REST && a.stride < 8) {
            const bool one = a.stride == 1;
            const int first = (lane & ~3) | (c & ((a.stride >> 1) - (one ? 0 : 1)));
            const float base0 = __shfl_sync(0xffffffffu, R[0][0], first);
            const float base1 = one ? base0 : __shfl_sync(0xffffffffu, R[0][1], first);
            const float part = 0.125f * static_cast<float>(a.stride);
            const float f0 = R[0][0] == base0 ? part : part * fast_exp2(R[0][0] - base0);
            const float f1 = R[0][1] == base1 ? part : part * fast_exp2(R[0][1] - base1);
            R[0][0] = base0;
            R[0][1] = base1;
            auto mean = [&](float& x0, float& x1) {
                x0 *= f0;
                x1 *= f1;
                if (one) x0 += x1;
                x0 += __shfl_xor_sync(0xffffffffu, x0, 2);
                if (!one) x1 += __shfl_xor_sync(0xffffffffu, x1, 2);
                if (a.stride <= 2) {
                    x0 += __shfl_xor_sync(0xffffffffu, x0, 1);
                    if (!one) x1 += __shfl_xor_sync(0xffffffffu, x1, 1);
                }
            };
            mean(l[0][0], l[0][1]);
#pragma unroll
            for (int k = 0; k < C::kNS; ++k) mean(zsum[0][k][0], zsum[0][k][1]);
#pragma unroll
            for (int b = 0; b < C::kSub; ++b)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    mean(acc[0][b][i][0], acc[0][b][i][1]);
                    mean(acc[0][b][i][2], acc[0][b][i][3]);
                }
        }

        // ---- the piece's state: to O, or to shared memory as acc[D], l, R per head
        const bool behind = !whole && !began_before;  // goes on behind the run: the ring is used up
        float* slot = behind ? reinterpret_cast<float*>(ring) : merge + warp * state_floats;
        if (behind) __syncwarp();
        if (!whole && lane == 0)
            cuts[2 * warp + (behind ? 1 : 0)] =
                CutUnit{cur.first(), cur.end(), cur.b * a.Hq + head0, nq};
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
                if (r >= nq) continue;
                const float inv = whole ? 1.0f / ls : 1.0f;
#pragma unroll
                for (int b = 0; b < C::kSub; ++b) {
                    const float z = zs[b * 32 / BS];
                    float4 v;  // elements element(b) + {0, 1, 2, 3}
                    v.x = fmaf(acc[t][b][0][j], 16777216.0f, z) * inv;
                    v.y = fmaf(acc[t][b][1][j], 1048576.0f, z) * inv;
                    v.z = fmaf(acc[t][b][0][j + 2], 16777216.0f, z) * inv;
                    v.w = fmaf(acc[t][b][1][j + 2], 1048576.0f, z) * inv;
                    if (whole)
                        store_out(a.o + (static_cast<long long>(cur.b) * a.Hq + head0 + r) * D + element(b),
                                  v, bf16);
                    else
                        *reinterpret_cast<float4*>(slot + r * C::kRecStride + element(b)) = v;
                }
                if (!whole && g == 0)
                    *reinterpret_cast<float2*>(slot + r * C::kRecStride + D) = make_float2(ls, R[t][j]);
            }
    }
    __syncthreads();

    // ---- join the states of the units that the CTA's warps cut.  A unit's first
    // state here is warp 0's first (it began before the CTA) or some warp's second;
    // the first states of the warps behind it follow while they are of the unit.
    // A warp joins a row; lane w knows warp w's descriptors.
    constexpr int kLanes = D / 4;  // lanes a row takes, 4 elements each
    constexpr int kSide = 32 / kLanes;
    const int i = lane % kLanes, side = lane / kLanes;
    const CutUnit before = cuts[0];
    const int first_of = lane < nw ? cuts[2 * lane].start : -1;
    const unsigned begins = __ballot_sync(0xffffffffu, lane < nw && cuts[2 * (lane % nw) + 1].start >= 0);
    const unsigned idle = __ballot_sync(0xffffffffu, first_of == -2);
    int turn = warp;  // rows go round the warps
    unsigned todo = begins;
    for (bool lead = before.start >= 0; lead || todo != 0; lead = false) {
        const int w = lead ? 0 : __ffs(todo) - 1;
        if (!lead) todo &= todo - 1;
        const CutUnit unit = lead ? before : cuts[2 * w + 1];
        const float* head = lead ? merge : reinterpret_cast<const float*>(smem + w * ring_bytes);
        const unsigned of_unit = __ballot_sync(0xffffffffu, first_of == unit.start);
        const int from = w + 1, count = __ffs(~((of_unit | idle) >> from)) - 1;
        const unsigned set = of_unit & (((1u << count) - 1u) << from);
        int r = turn;
        for (; r < unit.nq; r += nw) {
            // lane w: the state of warp w; lane 31: the first
            const bool have = lane == 31 || (set >> lane & 1u);
            float2 lr = make_float2(0.0f, -INFINITY);
            if (have)
                lr = *reinterpret_cast<const float2*>((lane == 31 ? head : merge + lane * state_floats) +
                                                      r * C::kRecStride + D);
            float m = lr.y;
#pragma unroll
            for (int off = 16; off; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
            const float f = lr.y == -INFINITY && lr.x == 0.0f ? 0.0f : fast_exp2(lr.y - m);
            float ls = lr.x * f;
#pragma unroll
            for (int off = 16; off; off >>= 1) ls += __shfl_xor_sync(0xffffffffu, ls, off);
            float4 v = *reinterpret_cast<const float4*>(head + r * C::kRecStride + 4 * i);
            float fw = __shfl_sync(0xffffffffu, f, 31);
            v.x *= fw, v.y *= fw, v.z *= fw, v.w *= fw;
#pragma unroll 4
            for (int k = from; k < from + count; ++k) {
                float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (set >> k & 1u)
                    x = *reinterpret_cast<const float4*>(merge + k * state_floats + r * C::kRecStride + 4 * i);
                fw = __shfl_sync(0xffffffffu, f, k);
                v.x = fmaf(x.x, fw, v.x);
                v.y = fmaf(x.y, fw, v.y);
                v.z = fmaf(x.z, fw, v.z);
                v.w = fmaf(x.w, fw, v.w);
            }
            if (side != 0) continue;
            if (unit.start >= g0 && unit.end <= g1) {
                const float inv = 1.0f / ls;
                store_out(a.o + static_cast<long long>(unit.row + r) * D + 4 * i,
                          make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv), bf16);
            } else {
                float* rec = a.recs + static_cast<long long>(cta * 2 + (unit.start >= g0 ? 1 : 0)) * state_floats +
                             r * C::kRecStride;
                __stcg(reinterpret_cast<float4*>(rec) + i, v);
                if (i == 0) __stcg(reinterpret_cast<float2*>(rec + D), make_float2(ls, m));
            }
        }
        turn = r - unit.nq;  // the rows of the next unit go on where these ended
    }

    // ---- units cut across CTAs: the one that began before (0), the one that goes
    // on behind (1); the last CTA to arrive at a unit's counter merges its records
    CutUnit behind;
    behind.start = -1;
    if (begins != 0) behind = cuts[2 * (31 - __clz(begins)) + 1];
    if (behind.start >= 0 && behind.end <= g1) behind.start = -1;
    if (before.start < 0 && behind.start < 0) return;
    // their first and last CTAs
    const unsigned before_first = before.start >= 0 ? cta_of(before.start) : 0;
    const unsigned before_last = before.end <= g1 ? cta : cta_of(before.end - 1);
    const unsigned behind_last = behind.start >= 0 ? cta_of(behind.end - 1) : 0;
    __syncthreads();
    if (threadIdx.x < 2) {
        const bool mine = (threadIdx.x == 0 ? before.start : behind.start) >= 0;
        const unsigned first = threadIdx.x == 0 ? before_first : cta;
        const unsigned last = threadIdx.x == 0 ? before_last : behind_last;
        unsigned done = 0;
        if (mine) {
            done = arrive_acq_rel(a.counters + first) == last - first;
            if (done) a.counters[first] = 0u;
        }
        flags[threadIdx.x] = done;
    }
    __syncthreads();
    const bool both = flags[0] && flags[1];
    if (!flags[0] && !flags[1]) return;
    // all warps merge the one unit, or half of them each of the two.  A warp takes
    // a row, or, with fewer rows than warps, a run of its pieces; the loads of 8
    // pieces (16 for D = 64) go out together.  How the pieces are grouped does not
    // depend on whether there is a second unit: sums keep their order.
    const int team = both ? nw >> 1 : nw;
    const int which = both ? (warp >= team ? 1 : 0) : (flags[0] ? 0 : 1);
    const int member = both && which ? warp - team : warp;
    const CutUnit unit = which == 0 ? before : behind;
    int log_split = 0;
    while ((unit.nq << (log_split + 1)) <= nw) ++log_split;
    const unsigned unit_first = which == 0 ? before_first : cta;
    const int np = static_cast<int>((which == 0 ? before_last : behind_last) - unit_first) + 1;
    const int rec_cta = 2 * state_floats;
    float* parts = which && both ? reinterpret_cast<float*>(smem) : merge;  // the rings are free
    float* rec0 = a.recs + static_cast<long long>(unit_first) * rec_cta;
    // the first CTA's piece is its second record, all others' the first
    auto at = [&](int p) { return rec0 + static_cast<long long>(p) * rec_cta + (p == 0 ? state_floats : 0); };
    for (int item = member; item < unit.nq << log_split; item += team) {
        const int r = item >> log_split, part = item - (r << log_split);
        const int pa = np * part >> log_split, pb = np * (part + 1) >> log_split;
        constexpr int kDeep = 8;
        float m = -INFINITY, ls = 0.0f;
        float4 v = make_float4(0, 0, 0, 0);
        for (int pw = pa; pw < pb; pw += kDeep * kSide) {
            float4 x[kDeep];
            float2 lr = make_float2(0.0f, -INFINITY);  // of piece pw + lane
            if (lane < kDeep * kSide && pw + lane < pb)
                lr = __ldcg(reinterpret_cast<const float2*>(at(pw + lane) + r * C::kRecStride + D));
#pragma unroll
            for (int k = 0; k < kDeep; ++k) {
                const int p = pw + k * kSide + side;
                x[k] = make_float4(0, 0, 0, 0);
                if (p < pb) x[k] = __ldcg(reinterpret_cast<const float4*>(at(p) + r * C::kRecStride) + i);
            }
            float top = lr.y;
#pragma unroll
            for (int off = 1; off < kDeep * kSide; off <<= 1)
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
            top = fmaxf(m, __shfl_sync(0xffffffffu, top, 0));
            const float old = m == top ? 1.0f : fast_exp2(m - top);
            m = top;
            const float f = lr.y == -INFINITY && lr.x == 0.0f ? 0.0f : fast_exp2(lr.y - m);
            ls = fmaf(ls, old, lr.x * f);
            v.x *= old, v.y *= old, v.z *= old, v.w *= old;
#pragma unroll
            for (int k = 0; k < kDeep; ++k) {
                const float fk = __shfl_sync(0xffffffffu, f, k * kSide + side);
                v.x = fmaf(x[k].x, fk, v.x);
                v.y = fmaf(x[k].y, fk, v.y);
                v.z = fmaf(x[k].z, fk, v.z);
                v.w = fmaf(x[k].w, fk, v.w);
            }
        }
#pragma unroll
        for (int off = 16; off; off >>= 1) ls += __shfl_xor_sync(0xffffffffu, ls, off);
        if constexpr (kSide == 2) {
            v.x += __shfl_xor_sync(0xffffffffu, v.x, 16);
            v.y += __shfl_xor_sync(0xffffffffu, v.y, 16);
            v.z += __shfl_xor_sync(0xffffffffu, v.z, 16);
            v.w += __shfl_xor_sync(0xffffffffu, v.w, 16);
        }
        if (side == 0) {
            float* dst = parts + item * C::kRecStride;
            *reinterpret_cast<float4*>(dst + 4 * i) = v;
            if (i == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(ls, m);
        }
    }
    __syncthreads();  // all records are read
    for (int r = member * kSide + side; r < unit.nq; r += team * kSide) {
        const float* src = parts + (r << log_split) * C::kRecStride;
        float4 v = *reinterpret_cast<const float4*>(src + 4 * i);
        float2 lr = *reinterpret_cast<const float2*>(src + D);
        for (int p = 1; p < 1 << log_split; ++p) {
            src += C::kRecStride;
            join(v, lr, *reinterpret_cast<const float4*>(src + 4 * i), *reinterpret_cast<const float2*>(src + D));
        }
        const float inv = 1.0f / lr.x;
        store_out(a.o + static_cast<long long>(unit.row + r) * D + 4 * i,
                  make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv), bf16);
    }
    // the records are zero again: nq * kRecStride floats of every piece
    for (int p = member; p < np; p += team) {
        float4* rec = reinterpret_cast<float4*>(at(p));
        for (int k = lane; k < unit.nq * C::kRecStride / 4; k += 32)
            __stcg(rec + k, make_float4(0, 0, 0, 0));
    }
}

}  // namespace tqkv
