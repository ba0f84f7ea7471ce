// tqkv_int4.cu — launch planning and C entry points of the 4-bit KV cache:
// writing, reading back, decode attention, and the head norms with the
// position rotation (kv_int4.cuh, decode_int4.cuh).

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <climits>
#include <cmath>
#include <cstdint>

#include "decode_int4.cuh"
#include "device_common.cuh"
#include "kv_int4.cuh"
#include "launch.h"
#include "tqkv.h"
#include "tqkv_internal.h"

namespace tqkv {

namespace {

constexpr int kMaxDevices = 64;

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

bool is_16bit(int dtype) { return dtype == TQKV_FP16 || dtype == TQKV_BF16; }

// SMs of the current device, looked up once.
cudaError_t current_sms(int* device, int* sms) {
    static std::atomic<int> known[kMaxDevices];
    cudaError_t e = cudaGetDevice(device);
    if (e != cudaSuccess) return e;
    if (*device < 0 || *device >= kMaxDevices) return cudaErrorInvalidDevice;
    int n = known[*device].load(std::memory_order_relaxed);
    if (n == 0) {
        e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, *device);
        if (e != cudaSuccess) return e;
        known[*device].store(n, std::memory_order_relaxed);
    }
    *sms = n;
    return cudaSuccess;
}

// Calls f(integral_constant D, integral_constant BS) for an accepted pair.
template <typename F>
tqkv_status for_shape(int D, int bs, F&& f) {
    using std::integral_constant;
    if (D == 64 && bs == 32) return f(integral_constant<int, 64>{}, integral_constant<int, 32>{});
    if (D == 64 && bs == 64) return f(integral_constant<int, 64>{}, integral_constant<int, 64>{});
    if (D == 128 && bs == 32) return f(integral_constant<int, 128>{}, integral_constant<int, 32>{});
    if (D == 128 && bs == 64) return f(integral_constant<int, 128>{}, integral_constant<int, 64>{});
    if (D == 128 && bs == 128) return f(integral_constant<int, 128>{}, integral_constant<int, 128>{});
    return TQKV_ERR_UNSUPPORTED;
}

template <int D>
unsigned rows_grid(long long rows, int unroll) {
    const long long per = (kInt4Threads / (D / 16)) * static_cast<long long>(unroll);
    return static_cast<unsigned>((rows + per - 1) / per);
}

tqkv_status make_rows(Int4Rows& g, int B, int H, int T, int S_cap, const int32_t* starts, int t0) {
    if (B <= 0 || H <= 0 || T <= 0 || S_cap <= 0 || T > S_cap) return TQKV_ERR_INVALID_SIZE;
    if (!starts && (t0 < 0 || static_cast<long long>(t0) + T > S_cap)) return TQKV_ERR_INVALID_SIZE;
    const long long BH = static_cast<long long>(B) * H;
    if (BH > INT_MAX / T) return TQKV_ERR_INVALID_SIZE;
    g.rows = static_cast<uint32_t>(BH * T);
    g.T = FastDiv(static_cast<uint32_t>(T));
    g.H = FastDiv(static_cast<uint32_t>(H));
    g.S_cap = S_cap;
    g.starts = starts;
    g.t0 = t0;
    g.sb = g.sh = g.st = 0;
    return TQKV_OK;
}

bool strides_ok(const long long* s) { return s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0; }

struct DecodePlan4 {
    int nt, rec_rows, slices;
    long long units, granules;  // granules at most: every sequence S rows long
    long long counted;          // granules that they and the units count for
};

DecodePlan4 plan_int4(int B, int Hq, int Hkv, int S) {
    DecodePlan4 p{};
    const int group = Hq / Hkv;
    // More than 8 heads share a pass of 16, where two passes of 8 would read the cache twice: B4 S131072
    // (heads of 128, bf16) takes 89.5 us with 64/4 heads and blocks of 128, 96.8 by two passes, and 95 with
    // 36/4 and blocks of 64, 115 by two.  A cache that L2 holds does not need it: 64/4 heads, 32 ragged
    // sequences of up to 4099 rows 26.6 and 26.4, one of 32769 rows 39.4 and 20.8.
    p.nt = group > 8 ? 2 : 1;
    p.rec_rows = group < 8 * p.nt ? group : 8 * p.nt;
    p.slices = (group + 8 * p.nt - 1) / (8 * p.nt);
    p.units = static_cast<long long>(B) * Hkv * p.slices;
    p.granules = p.units * ((static_cast<long long>(S) + kGranule - 1) / kGranule);
    p.counted = p.granules + p.units * kUnitCost;
    return p;
}

// One CTA an SM at most.  Without rows (S = 0) one writes the zeros and needs no workspace.
long long int4_grid(const DecodePlan4& p, int D, int sms, int warps) {
    if (p.granules == 0) return 1;
    return int4_ctas<long long>(p.counted, p.units, sms, warps * (4096 / D / kGranule));
}

size_t int4_counters(long long grid) { return (static_cast<size_t>(grid) * 4 + 255) / 256 * 256; }

// Counters and two records for every CTA.  For as many CTAs as any kernel may have with these or
// smaller sizes: the size grows with B, H_kv and S, so that a workspace for the largest batch
// serves every smaller one (int4_ctas alone does not: 149 units may take 75 CTAs, 148 take 148).
size_t int4_workspace(const DecodePlan4& p, int D, int sms) {
    const long long tiles = p.counted / (kI4MinWarps * (4096 / D / kGranule));
    const long long most = tiles > p.units ? tiles : p.units;
    const long long grid = p.granules == 0 ? 1 : most > sms ? sms : most;
    if (grid <= 1) return 0;
    return int4_counters(grid) + static_cast<size_t>(grid) * 2 * p.rec_rows * (D + 4) * sizeof(float);
}

template <int D, int BS, int NT, bool REST>
tqkv_status decode_int4_impl(Int4DecodeArgs a, const DecodePlan4& p, int bf16, void* workspace,
                             size_t workspace_bytes, cudaStream_t stream) {
    using C = I4Cfg<D, BS, NT, REST>;
    int dev = 0, sms = 0;
    cudaError_t e = current_sms(&dev, &sms);
    if (e != cudaSuccess) return from_cuda(e);
    auto fn = decode_int4_kernel<D, BS, NT, REST>;
    constexpr int kSmem = 227 * 1024;
    static std::atomic<bool> opted[kMaxDevices];
    if (!opted[dev].load(std::memory_order_acquire)) {
        e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
        if (e != cudaSuccess) return from_cuda(e);
        opted[dev].store(true, std::memory_order_release);
    }
    const long long grid = int4_grid(p, D, sms, C::kWarps);
    if (grid > 1 && (!workspace || workspace_bytes < int4_workspace(p, D, sms))) return TQKV_ERR_WORKSPACE;
    if (!aligned(workspace, 16)) return TQKV_ERR_MISALIGNED;
    a.counters = static_cast<unsigned int*>(workspace);
    a.recs = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) +
                                      int4_counters(grid));
    return from_cuda(launch_kernel_dependent(fn, dim3(static_cast<unsigned>(grid)), dim3(32 * C::kWarps),
                                             C::smem_bytes(p.rec_rows), stream, a, bf16));
}

}  // namespace
}  // namespace tqkv

using namespace tqkv;

extern "C" {

tqkv_status tqkv_kv_append_int4(const void* x, const long long* x_strides, uint8_t* cache_q,
                                void* cache_s, const int32_t* starts, int t0, int B, int H, int T,
                                int D, int block_size, int S_cap, int dtype, cudaStream_t stream) {
    if (!is_supported_int8(D, block_size) || !is_16bit(dtype)) return TQKV_ERR_UNSUPPORTED;
    Int4Rows g;
    const tqkv_status st = make_rows(g, B, H, T, S_cap, starts, t0);
    if (st != TQKV_OK) return st;
    if (!x || !cache_q || !cache_s) return TQKV_ERR_NULL;
    if (!aligned(x, 16) || !aligned(cache_q, 16) || !aligned(cache_s, 16) ||
        !aligned(starts, 4) || (x_strides && !strides_ok(x_strides)))
        return TQKV_ERR_MISALIGNED;
    g.st = x_strides ? x_strides[2] : D;
    g.sh = x_strides ? x_strides[1] : static_cast<long long>(T) * D;
    g.sb = x_strides ? x_strides[0] : static_cast<long long>(H) * T * D;
    return for_shape(D, block_size, [&](auto d, auto bs) {
        auto fn = dtype == TQKV_BF16 ? kv_append_int4_kernel<d(), bs(), true>
                                     : kv_append_int4_kernel<d(), bs(), false>;
        return from_cuda(launch_kernel_dependent(
            fn, dim3(rows_grid<d()>(g.rows, 1)), dim3(kInt4Threads), 0, stream,
            static_cast<const uint16_t*>(x), reinterpret_cast<uint32_t*>(cache_q),
            static_cast<uint32_t*>(cache_s), g));
    });
}

tqkv_status tqkv_kv_compress_int4(const void* x, uint8_t* xq, void* scales, int B, int H, int S,
                                  int D, int block_size, int dtype, cudaStream_t stream) {
    return tqkv_kv_append_int4(x, nullptr, xq, scales, nullptr, 0, B, H, S, D, block_size, S, dtype,
                               stream);
}

tqkv_status tqkv_kv_reconstruct_int4(const uint8_t* cache_q, const void* cache_s, void* y,
                                     const int32_t* starts, int t0, int B, int H, int T, int D,
                                     int block_size, int S_cap, int dtype, cudaStream_t stream) {
    if (!is_supported_int8(D, block_size) || !is_16bit(dtype)) return TQKV_ERR_UNSUPPORTED;
    Int4Rows g;
    const tqkv_status st = make_rows(g, B, H, T, S_cap, starts, t0);
    if (st != TQKV_OK) return st;
    if (!cache_q || !cache_s || !y) return TQKV_ERR_NULL;
    if (!aligned(cache_q, 16) || !aligned(cache_s, 16) || !aligned(y, 16) || !aligned(starts, 4))
        return TQKV_ERR_MISALIGNED;
    return for_shape(D, block_size, [&](auto d, auto bs) {
        auto fn = dtype == TQKV_BF16 ? kv_reconstruct_int4_kernel<d(), bs(), true>
                                     : kv_reconstruct_int4_kernel<d(), bs(), false>;
        return from_cuda(launch_kernel_dependent(
            fn, dim3(rows_grid<d()>(g.rows, kReadUnroll)), dim3(kInt4Threads), 0, stream,
            reinterpret_cast<const uint32_t*>(cache_q), static_cast<const uint32_t*>(cache_s),
            static_cast<uint4*>(y), g));
    });
}

size_t tqkv_decode_int4_workspace_bytes(int B, int H_q, int H_kv, int S, int D) {
    if (B <= 0 || H_q <= 0 || H_kv <= 0 || H_q % H_kv != 0 || S <= 0 || (D != 64 && D != 128))
        return 0;
    int dev = 0, sms = 0;
    if (current_sms(&dev, &sms) != cudaSuccess) return 0;
    const DecodePlan4 p = plan_int4(B, H_q, H_kv, S);
    return int4_workspace(p, D, sms);
}

tqkv_status tqkv_decode_int4(const void* q, const uint8_t* kq, const void* ks, const uint8_t* vq,
                             const void* vs, const int32_t* lengths, void* o, int B, int H_q,
                             int H_kv, int S, int S_cap, int D, int block_size, int dtype,
                             void* workspace, size_t workspace_bytes, cudaStream_t stream) {
    if (!is_supported_int8(D, block_size) || !is_16bit(dtype)) return TQKV_ERR_UNSUPPORTED;
    if (B <= 0 || H_q <= 0 || H_kv <= 0 || H_q % H_kv != 0 || S < 0 || S_cap <= 0 || S > S_cap)
        return TQKV_ERR_INVALID_SIZE;
    // rows are counted in 32 bits, in granules of 16
    if (static_cast<long long>(B) * H_q > INT_MAX || S > INT_MAX - 1024) return TQKV_ERR_INVALID_SIZE;
    if (!q || !o || !kq || !ks || !vq || !vs) return TQKV_ERR_NULL;
    if (!aligned(q, 16) || !aligned(o, 16) || !aligned(kq, 16) || !aligned(vq, 16) ||
        !aligned(ks, 16) || !aligned(vs, 16) || !aligned(lengths, 4))
        return TQKV_ERR_MISALIGNED;
    Int4DecodeArgs a{};
    a.q = static_cast<const uint16_t*>(q);
    a.kq = kq;
    a.vq = vq;
    a.ks = static_cast<const uint32_t*>(ks);
    a.vs = static_cast<const uint32_t*>(vs);
    a.o = static_cast<uint16_t*>(o);
    a.lengths = lengths;
    a.S_cap = S_cap;
    a.B = B;
    a.Hq = H_q;
    a.Hkv = H_kv;
    a.group = H_q / H_kv;
    a.S = S;
    a.score_scale = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(D)));
    const DecodePlan4 p = plan_int4(B, H_q, H_kv, S);
    if (p.granules + p.units * kUnitCost > INT_MAX) return TQKV_ERR_INVALID_SIZE;
    a.slices = p.slices;
    a.rec_rows = p.rec_rows;
    const int bf16 = dtype == TQKV_BF16;
    a.stride = 8;  // fp16: copies of the heads in the columns that a small group leaves idle, or rests
    while (!bf16 && a.stride / 2 >= a.group) a.stride /= 2;
    return for_shape(D, block_size, [&](auto d, auto bs) {
        auto run = [&](auto nt, auto rest) {
            return decode_int4_impl<d(), bs(), nt(), rest()>(a, p, bf16, workspace, workspace_bytes, stream);
        };
        using std::integral_constant;
        using std::bool_constant;
        if (p.nt == 2)
            return bf16 ? run(integral_constant<int, 2>{}, bool_constant<false>{})
                        : run(integral_constant<int, 2>{}, bool_constant<true>{});
        return bf16 || a.stride < 8 ? run(integral_constant<int, 1>{}, bool_constant<false>{})
                                    : run(integral_constant<int, 1>{}, bool_constant<true>{});
    });
}

static tqkv_status rope_checked(const tqkv_norm_rope_args* p, bool append, cudaStream_t stream) {
    if (!p) return TQKV_ERR_NULL;
    const int D = p->D, rot = p->rot_dim, axes = p->axes;
    if ((D != 64 && D != 128) || !is_16bit(p->dtype)) return TQKV_ERR_UNSUPPORTED;
    if (append && !is_supported_int8(D, p->block_size)) return TQKV_ERR_UNSUPPORTED;
    if (rot <= 0 || rot > D || rot % 16 != 0 || axes < 1 || axes > 4) return TQKV_ERR_UNSUPPORTED;
    long long sum = 0;
    for (int i = 0; i < axes; ++i) {
        if (p->sections[i] < 0) return TQKV_ERR_INVALID_SIZE;
        sum += p->sections[i];
    }
    if (axes > 1 && sum != rot / 2) return TQKV_ERR_INVALID_SIZE;
    if (p->B <= 0 || p->H_q <= 0 || p->H_kv <= 0 || p->T <= 0 || p->max_pos <= 0)
        return TQKV_ERR_INVALID_SIZE;
    if (!(p->eps >= 0.0)) return TQKV_ERR_INVALID_SIZE;
    const long long tokens = static_cast<long long>(p->B) * p->T;
    if (tokens > INT_MAX) return TQKV_ERR_INVALID_SIZE;
    if (append) {
        if (p->S_cap <= 0 || p->T > p->S_cap) return TQKV_ERR_INVALID_SIZE;
        if (!p->starts && (p->t0 < 0 || static_cast<long long>(p->t0) + p->T > p->S_cap))
            return TQKV_ERR_INVALID_SIZE;
    }
    if (!p->q || !p->k || !p->q_out || !p->table || !p->positions) return TQKV_ERR_NULL;
    if (append ? (!p->v || !p->kq || !p->ks || !p->vq || !p->vs) : !p->k_out) return TQKV_ERR_NULL;
    if (!aligned(p->q, 16) || !aligned(p->k, 16) || !aligned(p->q_out, 16) ||
        !aligned(p->q_weight, 16) || !aligned(p->k_weight, 16) || !aligned(p->table, 16) ||
        !aligned(p->positions, 4) || !aligned(p->starts, 4) || !strides_ok(p->q_strides) ||
        !strides_ok(p->k_strides))
        return TQKV_ERR_MISALIGNED;
    if (append ? (!aligned(p->v, 16) || !strides_ok(p->v_strides) || !aligned(p->kq, 16) ||
                  !aligned(p->ks, 16) || !aligned(p->vq, 16) || !aligned(p->vs, 16))
               : !aligned(p->k_out, 16))
        return TQKV_ERR_MISALIGNED;

    int dev = 0, sms = 0;
    const cudaError_t e = current_sms(&dev, &sms);
    if (e != cudaSuccess) return from_cuda(e);
    RopeArgs a{};
    a.q = static_cast<const uint16_t*>(p->q);
    a.k = static_cast<const uint16_t*>(p->k);
    a.v = static_cast<const uint16_t*>(p->v);
    a.q_sb = p->q_strides[0], a.q_sh = p->q_strides[1], a.q_st = p->q_strides[2];
    a.k_sb = p->k_strides[0], a.k_sh = p->k_strides[1], a.k_st = p->k_strides[2];
    a.v_sb = p->v_strides[0], a.v_sh = p->v_strides[1], a.v_st = p->v_strides[2];
    a.q_out = static_cast<uint16_t*>(p->q_out);
    a.k_out = static_cast<uint16_t*>(p->k_out);
    a.q_w = static_cast<const uint16_t*>(p->q_weight);
    a.k_w = static_cast<const uint16_t*>(p->k_weight);
    a.table = reinterpret_cast<const float2*>(p->table);
    a.pos = p->positions;
    a.kc = reinterpret_cast<uint32_t*>(p->kq);
    a.kp = static_cast<uint32_t*>(p->ks);
    a.vc = reinterpret_cast<uint32_t*>(p->vq);
    a.vp = static_cast<uint32_t*>(p->vs);
    a.starts = p->starts;
    a.eps = p->eps;
    a.S_cap = p->S_cap;
    a.tokens = static_cast<uint32_t>(tokens);
    a.Hq = p->H_q, a.Hkv = p->H_kv, a.T = p->T, a.t0 = p->t0;
    a.max_pos = p->max_pos, a.rot = rot, a.axes = axes;
    a.s1 = axes > 1 ? p->sections[0] : INT_MAX;
    a.s2 = axes > 2 ? a.s1 + p->sections[1] : INT_MAX;
    a.s3 = axes > 3 ? a.s2 + p->sections[2] : INT_MAX;
    const int heads = 512 / D;  // a warp's step
    a.q_steps = (p->H_q + heads - 1) / heads;
    a.kv_steps = (p->H_kv + heads - 1) / heads;
    const int steps = a.q_steps + (append ? 2 : 1) * a.kv_steps;
    const long long all = tokens * steps;
    if (all > INT_MAX) return TQKV_ERR_INVALID_SIZE;
    const int warps_per_cta = kInt4Threads / 32;
    const long long resident = static_cast<long long>(sms) * kRopeCtas * warps_per_cta;
    a.warps = static_cast<uint32_t>(all < resident ? all : resident);
    a.run = static_cast<uint32_t>(all) / a.warps;
    a.longer = static_cast<uint32_t>(all) - a.run * a.warps;
    a.steps = FastDiv(static_cast<uint32_t>(steps));
    a.divT = FastDiv(static_cast<uint32_t>(p->T));
    const unsigned grid = (a.warps + warps_per_cta - 1) / warps_per_cta;
    const bool bf16 = p->dtype == TQKV_BF16, inter = p->interleaved != 0;
    auto launch = [&](auto fn) {
        return from_cuda(launch_kernel_dependent(fn, dim3(grid), dim3(kInt4Threads), 0, stream, a));
    };
    if (!append) {
        if (D == 64)
            return bf16 ? (inter ? launch(qk_norm_rope_kernel<64, 32, true, false, true>)
                                 : launch(qk_norm_rope_kernel<64, 32, true, false, false>))
                        : (inter ? launch(qk_norm_rope_kernel<64, 32, false, false, true>)
                                 : launch(qk_norm_rope_kernel<64, 32, false, false, false>));
        return bf16 ? (inter ? launch(qk_norm_rope_kernel<128, 32, true, false, true>)
                             : launch(qk_norm_rope_kernel<128, 32, true, false, false>))
                    : (inter ? launch(qk_norm_rope_kernel<128, 32, false, false, true>)
                             : launch(qk_norm_rope_kernel<128, 32, false, false, false>));
    }
    return for_shape(D, p->block_size, [&](auto d, auto bs) {
        return bf16 ? (inter ? launch(qk_norm_rope_kernel<d(), bs(), true, true, true>)
                             : launch(qk_norm_rope_kernel<d(), bs(), true, true, false>))
                    : (inter ? launch(qk_norm_rope_kernel<d(), bs(), false, true, true>)
                             : launch(qk_norm_rope_kernel<d(), bs(), false, true, false>));
    });
}

tqkv_status tqkv_qk_norm_rope(const tqkv_norm_rope_args* args, cudaStream_t stream) {
    return rope_checked(args, false, stream);
}

tqkv_status tqkv_qk_norm_rope_append_int4(const tqkv_norm_rope_args* args, cudaStream_t stream) {
    return rope_checked(args, true, stream);
}

}  // extern "C"
