// Device helpers of the paged operators (pages.cu): value types, the ragged batch, pages and key
// ranges.
#pragma once

#include <atomic>
#include <cfloat>
#include <type_traits>

#include <cuda_bf16.h>

#include "kernels.cuh"

namespace sp {

// ---- value types -------------------------------------------------------------------------------
SP_DEVINL float to_float(float v) { return v; }
SP_DEVINL float to_float(__half v) { return __half2float(v); }
SP_DEVINL float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
SP_DEVINL T from_float(float v) {
    if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __float2bfloat16_rn(v);
    else return v;
}
// two values as one 32-bit word, a in the low half
template <typename T>
SP_DEVINL uint32_t pack2(float a, float b) {
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}
template <typename T>
SP_DEVINL void unpack2(uint32_t w, float &a, float &b) {
    if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
        a = f.x;
        b = f.y;
    } else {
        a = __uint_as_float(w << 16);
        b = __uint_as_float(w & 0xffff0000u);
    }
}
SP_DEVINL float exp2_approx(float x) {                       // 2^x, relative error below 2^-22; 2^-inf = 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// A row's (or a key range's) statistics: m, its largest q k before the scale, and l, the sum of 2^((q k - m) c), c = scale
// log2(e). The difference is taken before the product: it is 0 at the maximum, however large the scores are (a rounded
// m c leaves up to 2^-24 of itself there).
// The log-sum-exp; no sum: no key. A row of NaN scores has a sum (NaN), but no maximum
SP_DEVINL float row_lse(float m, float l, float c) {
    return l == 0.f ? -INFINITY : fmaf(m, c, log2f(l)) * 0.6931471805599453f;
}
SP_DEVINL float row_scale(const PagesAttention &p) { return fminf(p.scale * 1.4426950408889634f, FLT_MAX); }
// c of a row whose queries were divided by `up`: never 0 or infinite (times -inf, or times 0 at the maximum, NaN). The
// divided row's scores are below 2^40, so that the least normal number leaves nothing of them
SP_DEVINL float row_scale(const PagesAttention &p, float up) { return fminf(fmaxf(row_scale(p) * up, FLT_MIN), FLT_MAX); }

// fp32 queries are split into fp16 halves after a power of two, exact to take back, that brings the row's largest |q| into
// [2^14, 2^15): any finite query has halves then, and what the lo half rounds off is 2^-39 of the largest
SP_DEVINL void row_power(float top, float &down, float &up) {
    const int e = min(max((int)(__float_as_uint(top) >> 23), 28), 254) - 141;
    down = __uint_as_float((uint32_t)(127 - e) << 23);
    up = __uint_as_float((uint32_t)(127 + e) << 23);
}

// ---- the ragged batch --------------------------------------------------------------------------
SP_DEVINL void set_status(int *status) {
    if (status) atomicCAS(status, 0, kErrPages);
}
SP_DEVINL int request_start(const PageBatchView &ba, int b) {
    return ba.q_start ? min(max(ba.q_start[b], 0), ba.T) : (int)min((long long)b * ba.max_q, (long long)ba.T);
}
// rows of the call: q_start's last, within the host's bound
SP_DEVINL int total_rows(const PageBatchView &ba) {
    return ba.q_start ? min(ba.T, ba.q_start[ba.B]) : (int)min((long long)ba.T, (long long)ba.B * ba.max_q);
}
// The request of row t < q_start[B] (the last b with q_start[b] <= t), by the whole warp: 32 probes a
// round.
SP_DEVINL int find_request(const PageBatchView &ba, int t, int lane) {
    if (!ba.q_start) return t / ba.max_q;
    int lo = 0, n = ba.B;
    while (n > 1) {
        const int step = (n + 31) / 32, at = lane * step;
        const bool le = at < n && ba.q_start[lo + at] <= t;
        const int c = max(0, __popc(__ballot_sync(0xffffffffu, le)) - 1) * step;
        lo += c;
        n = min(step, n - c);
    }
    return lo;
}
// a request's own keys, within its table
SP_DEVINL int own_len(const PagesAttention &p, int b, int lane) {
    const int len = p.ba.lens[b];
    const long long cap = (long long)p.ba.table_width * p.pg.page_size;
    if (len < 0 || len > cap) {
        if (lane == 0) set_status(p.pg.status);
        return len < 0 ? 0 : (int)cap;
    }
    return len;
}
// ---- key ranges --------------------------------------------------------------------------------
constexpr int kPagesGrain = 128;                             // key ranges are multiples of this
constexpr int kPagesOwnKeys = 256;                           // own keys per range at least
constexpr int kPagesMaxSplits = 32;
struct PagesPlan {
    // all rows over ranges of the prefix, each request's rows over ranges of its own keys: row tiles x key
    // ranges; `tc`: k_pages_tc (else k_pages_rows); `alt`: its two groups of warps take alternate key tiles
    // of one row tile and leave a partial each
    int prefix_tiles, prefix_splits, prefix_chunk, prefix_slots, prefix_tc, prefix_alt;
    int own_tiles, own_splits, own_tc, own_alt;
    int whole;                                               // own_tiles over the prefix and the own keys, no partials
                                                             // (own_tc: by k_pages_tc, else by k_pages_rows)
    int slots;                                               // partials per (token, head); 1: no merge
    float *acc, *ml;                                         // [slots][T][heads][hd], [slots][T][heads][m, l]
};
// a request's own keys in at most `most` ranges of `chunk` keys (the same in every kernel)
SP_DEVINL void own_chunks(int len, int most, int &chunk, int &n) {
    const int want = max(1, min(most, (len + kPagesOwnKeys - 1) / kPagesOwnKeys));
    chunk = max(kPagesGrain, ((len + want - 1) / want + kPagesGrain - 1) / kPagesGrain * kPagesGrain);
    n = max(1, (len + chunk - 1) / chunk);                   // no key: one empty range
}

// pages_tc.cu
bool pages_tc_fits(const PagesView &pg);
cudaError_t launch_pages_tc(const PagesAttention &p, const PagesPlan &pl, cudaStream_t s);

// Raise a kernel's dynamic shared memory limit, once per device and kernel.
template <typename... KArgs>
cudaError_t raise_smem(void (*kernel)(KArgs...), int bytes) {
    static std::atomic<const void *> done[64][32];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    for (int i = 0; i < 32; ++i)
        if (done[dev & 63][i].load() == reinterpret_cast<const void *>(kernel)) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
    for (int i = 0; i < 32; ++i) {
        const void *none = nullptr;
        if (done[dev & 63][i].compare_exchange_strong(none, reinterpret_cast<const void *>(kernel))) break;
    }
    return cudaSuccess;
}

// Launch a kernel that may start while the one before it in the stream finishes (programmatic dependent
// launch): it waits (griddepcontrol.wait) before it reads what that one wrote, or before it ends.
template <typename... KArgs, typename... Args>
cudaError_t launch_dependent(void (*kernel)(KArgs...), dim3 grid, int block, size_t smem, cudaStream_t s, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

}  // namespace sp
