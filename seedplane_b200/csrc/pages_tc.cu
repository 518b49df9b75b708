// Attention of many rows over pages on the 5th-generation tensor cores, sm_100a: the shared prefix under the
// stacked rows of a whole batch, and requests that bring many tokens (sp_pages_attention).
//
// A CTA takes up to 256 (token, head) rows of one kv head's group and walks a key sequence (a range of the
// prefix, or the prefix and then one request's own keys) in tiles of 128 keys:
//   S_q = Q_q K^T    tcgen05.mma M 128, N 128 into TMEM (two row tiles q, 128 columns each)
//   P_q = 2^((S - m) c + bias), m the row's running maximum, kept while it grows by less than 2^8 (2^4 with fp32
//         queries), so that the sums and O seldom need rescaling (P <= 2^15 then, within either 16-bit type's range);
//         written over S_q in TMEM in the cache's type
//   O_q += P_q V     tcgen05.mma with A = P_q in TMEM, B = V as it lies in its pages (MN-major)
// Packed prompts (12 requests, 3,679 rows x 28 heads over 3,001 + 560 keys) take 199 us, 898 TFLOP/s, at the 1,000 W
// cap (1.8 GHz); the MMAs alone take 127 us, with the tiles' loads 151, the softmax with the loads 176 (before the
// exponents took their differences first, 2.5 us in all). A row tile's
// steps follow one another, so two row tiles take turns:
//   warps 0-7, 8-15  one row tile each, two threads a row with 64 columns each: tcgen05.ld of the scores, maximum,
//                    exponentials (in fp32, base 2), tcgen05.st in place (one thread a row and 128 registers of
//                    scores was 5 % slower for decode steps, 2 % faster for prompts)
//   warp 16          TMA of the pages' rows (64 dims x a page's slots a box, 128-byte swizzle) into a ring
//   warp 17          issues the MMAs: while one row tile's scores are exponentiated, the other's products run
// One row tile alone (at most 128 rows: a small batch, or fp32 queries) gives both groups of warps work by
// taking alternate key tiles, each with its own (m, l, O); their partials are joined like those of key ranges.
// fp32 queries: Q as fp16 hi and lo tiles, S = Qlo K^T + Qhi K^T, P as hi and lo, O += Plo V + Phi V. The MMAs cut off
// what they add to an accumulator, 2^-24 of it an addition: the small products go first (S: 3.7e-6 -> 2.4e-6 of the
// result after 32,768 keys), and every kTcFlush tiles O is added to a second set of columns with ordinary rounding
// (3,100 keys at once: 8e-6; every 4 tiles 1.6e-6, every 2 1.1e-6). Two groups that share a row tile have no
// columns to spare: their key ranges are kept short instead.
// Slots of a page behind the last key may hold anything: their scores are replaced, their V rows zeroed in
// shared memory (0 x NaN would reach O). Every wait is bounded.
#include <cuda.h>

#include <algorithm>
#include <cmath>

#include "pages.cuh"
#include "tc.cuh"

namespace sp {

namespace {

constexpr int kTcKeys = 128;                 // keys of a tile
constexpr int kTcRows = 128;                 // rows of a row tile
constexpr int kTcSoftmax = 512;              // threads: two row tiles x two halves of the columns x 128 rows
constexpr int kTcThreads = kTcSoftmax + 64;
constexpr int kTcProducer = 16, kTcMma = 17; // warps
constexpr int kTcStages = 4;
constexpr uint32_t kTcSpin = 1u << 22;
constexpr int kTcFlush = 2;                  // fp32 queries: O is added up in fp32 outside the MMAs every so many tiles
// A row's probabilities are held times 2^kTcBias, and its running maximum may lag behind by kTcGrow (in base 2). In fp16
// they end at 2^15, and its subnormals' rounding, 2^-25, lies kTcBias further below the maximum: without
// it many small weights behind a large one (a key that takes most of the weight and has a value near 0) lose their bits.
// A shorter lag means a longer bias and more rescaling: none for fp16 queries (prompts 196 us, with a lag of 4 207), but
// fp32 ones carry a lo half too (3,679 rows 465 us with a lag of 8, 481 with 4, 490 with 2). bf16 has fp32's range.
template <typename TQ, typename TC>
constexpr float kTcGrow = std::is_same<TC, __half>::value && sizeof(TQ) == 4 ? 4.0f : 8.0f;
template <typename TQ, typename TC>
constexpr float kTcBias = std::is_same<TC, __half>::value ? 15.0f - kTcGrow<TQ, TC> : 0.0f;

template <int HD>
struct TcSmem {
    static constexpr int kHalf = kTcKeys * 128;              // 64 dims of 128 rows
    static constexpr int kTile = kHalf * (HD / 64);          // a K, V or Q tile
    static constexpr int kQ = 2 * kTile;                     // two row tiles, or hi and lo
    static constexpr int kBytes = kQ + kTcStages * kTile + 1024;
};

SP_DEVINL void tma_page(uint32_t dst, const CUtensorMap *map, int d, int slot, int head, int page, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(d), "r"(slot), "r"(head), "r"(page), "r"(smem_u32(bar))
        : "memory");
}
// V rows as the B operand: dims contiguous (MN-major), 64 dims a 128-byte row, 8 keys a swizzle atom; the
// next 64 dims lie kHalf bytes on, the next 8 keys 1,024.
SP_DEVINL uint64_t v_desc(uint32_t addr, uint32_t half) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(half >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}
// A from TMEM (16-bit values, two a column)
SP_DEVINL void mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n"
        ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate));
}
SP_DEVINL void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]));
}
// Two fp32 values as one 64-bit operand of the packed instructions.
SP_DEVINL uint64_t f2(float a, float b) { return (uint64_t)__float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32); }
SP_DEVINL float f2_lo(uint64_t v) { return __uint_as_float((uint32_t)v); }
SP_DEVINL float f2_hi(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }
SP_DEVINL uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
SP_DEVINL uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
SP_DEVINL float max3(float a, float b, float c) {             // NaN is passed over, as by fmaxf
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
SP_DEVINL void st_shared16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
SP_DEVINL bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
SP_DEVINL void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Instruction descriptor: D fp32, A and B of the cache's type, M 128, N = n; B MN-major or K-major.
template <typename TC>
SP_DEVINL constexpr uint32_t tc_idesc(int n, bool mn) {
    const uint32_t fmt = std::is_same<TC, __half>::value ? 0u : 1u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | ((mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

struct TcBarriers {
    uint64_t full[kTcStages], empty[kTcStages];
    uint64_t q_full, s_full[2], p_full[2], o_full[2], tail, drain;
};

// The keys an item walks: tiles [0, n_a) of the first segment, then [n_a, n) of the second.
struct TcKeys {
    const int *table_a, *table_b;
    int lo_a, hi_a, hi_b;                    // first segment [lo_a, hi_a), second [0, hi_b)
    int n_a, n;
    SP_DEVINL int lo(int i) const { return i < n_a ? lo_a + i * kTcKeys : (i - n_a) * kTcKeys; }
    SP_DEVINL int hi(int i) const { return i < n_a ? hi_a : hi_b; }
    SP_DEVINL const int *table(int i) const { return i < n_a ? table_a : table_b; }
};

struct TcWait {
    volatile int *abort;
    int *status;
    SP_DEVINL bool wait(uint64_t *bar, uint32_t parity) const {
        for (uint32_t i = 0; i < kTcSpin; ++i) {
            if (mbar_try_wait(bar, parity)) return true;
            if ((i & 127u) == 127u && *abort) return false;
        }
        *abort = 1;
        if (status) atomicCAS(status, 0, kErrMbarTimeout);
        return false;
    }
    // by a whole warp: the same answer in every lane
    SP_DEVINL bool wait_warp(uint64_t *bar, uint32_t parity) const { return __all_sync(0xffffffffu, wait(bar, parity)); }
};

template <int HD, typename TQ, typename TC>
__global__ void __launch_bounds__(kTcThreads, 1)
    k_pages_tc(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, PagesAttention p,
               PagesPlan pl) {
    constexpr bool kSplit = sizeof(TQ) == 4;
    using L = TcSmem<HD>;
    constexpr int CH = HD / 8, KS = HD / 16;
    extern __shared__ uint8_t tc_smem_raw[];
    __shared__ __align__(8) TcBarriers bar;
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    __shared__ float s_swap[2][2][kTcRows];
    __shared__ float s_up[kSplit ? kTcRows : 1];             // what a row's queries were divided by
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const PageBatchView &ba = p.ba;
    const int g = blockIdx.y, G = p.nh / p.pg.nkv;
    griddep_launch_dependents();
    if (warp == kTcProducer && lane == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tm_k)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tm_v)) : "memory");
    }
    // the item
    const int total = total_rows(ba);
    int q0 = 0, row0, nrows, slot = 0, own0 = INT_MAX / 2, own_tile0 = INT_MAX, item = blockIdx.x;
    bool alt = false;                        // the groups of warps take alternate key tiles of one row tile
    TcKeys ks{};
    const int n_prefix = pl.prefix_tc ? pl.prefix_tiles * pl.prefix_splits : 0;
    if (item < n_prefix) {                   // all rows over a range of the prefix
        alt = pl.prefix_alt;
        const int z = item / pl.prefix_tiles, tile_rows = alt ? kTcRows : 2 * kTcRows;
        row0 = (item - z * pl.prefix_tiles) * tile_rows;
        nrows = min(tile_rows, total * G - row0);
        slot = z << pl.prefix_alt;
        ks.table_a = ba.prefix;
        ks.lo_a = z * pl.prefix_chunk;
        ks.hi_a = min(ba.prefix_len, ks.lo_a + pl.prefix_chunk);
        ks.n = ks.n_a = (ks.hi_a - ks.lo_a + kTcKeys - 1) / kTcKeys;
        if (nrows <= 0) return;
    } else {                                 // a request's rows over its own keys, or the prefix and them
        alt = pl.own_alt;
        item -= n_prefix;
        const int per = pl.own_tiles * (pl.whole ? 1 : pl.own_splits), b = item / per;
        item -= b * per;
        const int z = item / pl.own_tiles, tile_rows = alt || kSplit ? kTcRows : 2 * kTcRows;
        row0 = (pl.own_tiles - 1 - (item - z * pl.own_tiles)) * tile_rows;    // the longest first
        q0 = request_start(ba, b);
        const int qn = min(request_start(ba, b + 1), total) - q0, len = own_len(p, b, tid);
        if (qn > ba.max_q && tid == 0) set_status(p.pg.status);
        nrows = min(tile_rows, qn * G - row0);
        if (nrows <= 0) return;
        own0 = len - qn;
        const int last = max(0, min(len, own0 + (row0 + nrows - 1) / G + 1));
        const int *table = ba.tables + (long long)b * ba.table_stride;
        if (pl.whole) {
            ks.table_a = ba.prefix;
            ks.hi_a = ba.prefix_len;
            ks.table_b = table;
            ks.hi_b = last;
            ks.n_a = (ks.hi_a + kTcKeys - 1) / kTcKeys;
            ks.n = ks.n_a + (last + kTcKeys - 1) / kTcKeys;
            own_tile0 = ks.n_a;
        } else {
            int chunk, parts;
            own_chunks(len, pl.own_splits, chunk, parts);
            slot = pl.prefix_slots + (z << pl.own_alt);
            if (z >= parts) {                // no such range: nothing to join
                for (int i = tid; i < nrows << pl.own_alt; i += kTcThreads) {
                    const int k = i / nrows, row = row0 + i - k * nrows;
                    const long long at = ((long long)(slot + k) * ba.T + q0 + row / G) * p.nh + g * G + row % G;
                    *reinterpret_cast<float2 *>(pl.ml + at * 2) = make_float2(-INFINITY, 0.f);
                }
                return;
            }
            ks.table_a = table;
            ks.lo_a = z * chunk;
            ks.hi_a = min(ks.lo_a + chunk, last);
            ks.n = ks.n_a = max(0, (ks.hi_a - ks.lo_a + kTcKeys - 1) / kTcKeys);
            own_tile0 = 0;
        }
    }
    const int n = ks.n;
    const int nq = alt || nrows > kTcRows ? 2 : 1;           // groups of softmax warps at work
    const uint32_t base = (smem_u32(tc_smem_raw) + 1023u) & ~1023u, ring = base + L::kQ;
    const TcWait w{&s_abort, p.pg.status};

    if (tid == 0) {
        s_abort = 0;
        for (int i = 0; i < kTcStages; ++i) {
            mbar_init(&bar.full[i], 1);
            mbar_init(&bar.empty[i], 1);
        }
        mbar_init(&bar.q_full, kTcSoftmax / 32);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar.s_full[i], 1);
            mbar_init(&bar.p_full[i], kTcSoftmax / 64);
            mbar_init(&bar.o_full[i], 1);
        }
        mbar_init(&bar.tail, 1);
        mbar_init(&bar.drain, 1);
        fence_mbar_init();
    }
    if (warp == kTcMma) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512u));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;

    if (warp == kTcProducer) {
        // ring order: K of the first `lead` tiles, then V of tile i and K of tile i + lead
        const int lead = alt ? 2 : 1;
        int it = 0, tails = 0;
        // the page numbers around K's and V's places in the sequence, 32 at a time: a tile's are at hand before
        // its stage is free
        struct Window {
            int pages, first = INT_MIN, seg = -1;
        } win_k, win_v;
        const auto load = [&](int i, bool is_v, Window &win) -> bool {
            const int st = it % kTcStages, lo = ks.lo(i), hi = ks.hi(i), keys = min(kTcKeys, hi - lo);
            const int per = min(p.pg.page_size, kTcKeys), pages = (keys + per - 1) / per;
            const int seg = i >= ks.n_a, first = lo / p.pg.page_size;
            if (seg != win.seg || first < win.first || first + (pages - 1) * per / p.pg.page_size > win.first + 31) {
                win.seg = seg;
                win.first = first;
                const int pi = first + lane;
                win.pages = (long long)pi * p.pg.page_size < hi ? __ldg(ks.table(i) + pi) : 0;
            }
            // lane: box `lane` of the tile (a page, or 128 slots of a larger one)
            const int key = lo + min(lane, pages - 1) * per, pi = key / p.pg.page_size;
            int page = __shfl_sync(0xffffffffu, win.pages, pi - win.first);
            const int slot0 = key - pi * p.pg.page_size;
            if ((unsigned)page >= (unsigned)p.pg.n_pages) {
                if (lane < pages) set_status(p.pg.status);
                page = p.pg.n_pages;         // outside the tensor: zeros
            }
            if (it >= kTcStages && !w.wait_warp(&bar.empty[st], (uint32_t)(it / kTcStages - 1) & 1u)) return false;
            const uint32_t dst = ring + (uint32_t)st * L::kTile;
            const bool tail = is_v && keys < kTcKeys;
            uint64_t *b = tail ? &bar.tail : &bar.full[st];
            if (lane == 0) mbar_arrive_expect_tx(b, (uint32_t)(pages * per) * HD * 2);
            __syncwarp();
            if (lane < pages) {
#pragma unroll
                for (int h = 0; h < HD / 64; ++h)
                    tma_page(dst + h * L::kHalf + lane * per * 128, is_v ? &tm_v : &tm_k, 64 * h, slot0, g, page, b);
            }
            __syncwarp();
            if (tail) {                      // rows behind the last key: zero, once the page's slots are there
                if (!w.wait_warp(&bar.tail, (uint32_t)tails++ & 1u)) return false;
                for (int r = keys * CH + lane; r < kTcKeys * CH; r += 32) {
                    const int row = r / CH, c = r - row * CH;
                    asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(dst + (c >> 3) * L::kHalf + row * 128 + (c & 7) * 16), "r"(0u)
                                 : "memory");
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar.full[st]);
            }
            ++it;
            return true;
        };
        int kc = 0, vc = 0;
        for (bool ok = true; ok && vc < n;) {
            const bool is_v = kc >= n || kc >= vc + lead;
            ok = is_v ? load(vc, true, win_v) : load(kc, false, win_k);
            ++(is_v ? vc : kc);
        }
        // no copy is in flight when the CTA ends, whoever gave up
        for (int j = max(0, it - kTcStages); j < it; ++j)
            for (uint32_t k = 0; k < kTcSpin && !mbar_try_wait(&bar.full[j % kTcStages], (uint32_t)(j / kTcStages) & 1u); ++k) {
            }
    } else if (warp == kTcMma) {
        // the whole warp runs the loop, one elected lane issues: control flow and descriptors stay uniform
        if (n > 0 && w.wait_warp(&bar.q_full, 0)) {
            constexpr uint32_t id_s = tc_idesc<TC>(kTcKeys, false), id_o = tc_idesc<TC>(HD, true);
            int it = 0;
            bool ok = true;
            int k_st = 0, v_st = 0;
            uint32_t p_ph[2] = {0u, 0u};
            const auto arrive = [&](int &st) {               // the ring's next tile
                st = it % kTcStages;
                ok = w.wait_warp(&bar.full[st], (uint32_t)(it / kTcStages) & 1u);
                ++it;
                tc_fence_after();
                return ok;
            };
            const auto commit = [&](uint64_t *b) {
                if (elect_one()) mma_commit(b);
                __syncwarp();
            };
            const auto scores = [&](int q) {                 // S_q = Q K^T
                const uint64_t kd = smem_desc_sw128(ring + (uint32_t)k_st * L::kTile, 1024);
                const uint64_t qd = smem_desc_sw128(base + (uint32_t)(kSplit || alt ? 0 : q) * L::kTile, 1024);
                if (elect_one()) {
#pragma unroll
                    for (int part = kSplit ? 1 : 0; part >= 0; --part)    // the small products first
#pragma unroll
                        for (int kk = 0; kk < KS; ++kk) {
                            const int o = ((kk >> 2) * L::kHalf + (kk & 3) * 32) >> 4;
                            mma_f16_id(tmem + 128 * q, qd + o + ((part * L::kTile) >> 4), kd + o, id_s, (kSplit && part == 0) || kk > 0);
                        }
                    mma_commit(&bar.s_full[q]);
                }
                __syncwarp();
            };
            const auto values = [&](int q, bool first) -> bool {                      // O_q += P_q V
                const uint64_t vd = v_desc(ring + (uint32_t)v_st * L::kTile, L::kHalf);
                if (!w.wait_warp(&bar.p_full[q], p_ph[q])) return ok = false;
                p_ph[q] ^= 1u;
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int part = kSplit ? 1 : 0; part >= 0; --part)
#pragma unroll
                        for (int kk = 0; kk < kTcKeys / 16; ++kk)
                            mma_ts(tmem + 256 + 128 * q, tmem + 128 * q + 32 * (kk >> 1) + 8 * (kk & 1) + 16 * part, vd + ((kk * 2048) >> 4), id_o,
                                   !(first && part == (kSplit ? 1 : 0) && kk == 0));
                }
                __syncwarp();
                return true;
            };
            if (alt) {
                for (int i = 0; i < 2 && i < n && ok; ++i) {
                    if (!arrive(k_st)) break;
                    scores(i);
                    commit(&bar.empty[k_st]);
                }
                for (int i = 0; i < n && ok; ++i) {
                    // the tiles are waited for before the probabilities: only those are on the chain of waits
                    if (!arrive(v_st) || (i + 2 < n && !arrive(k_st)) || !values(i & 1, i < 2)) break;
                    commit(&bar.empty[v_st]);
                    if (i + 2 < n) {
                        scores(i & 1);
                        commit(&bar.empty[k_st]);
                    } else {
                        commit(&bar.o_full[i & 1]);
                    }
                }
            } else {
                if (arrive(k_st)) {
                    for (int q = 0; q < nq; ++q) scores(q);
                    commit(&bar.empty[k_st]);
                }
                for (int i = 0; i < n && ok; ++i) {
                    for (int q = 0; q < nq && ok; ++q) {
                        if (q == 0 && (!arrive(v_st) || (i + 1 < n && !arrive(k_st)))) break;
                        if (!values(q, i % (kSplit ? kTcFlush : INT_MAX) == 0)) break;
                        if (q == nq - 1) commit(&bar.empty[v_st]);
                        if (i + 1 < n) {
                            scores(q);
                            if (q == nq - 1) commit(&bar.empty[k_st]);
                        } else {
                            commit(&bar.o_full[q]);
                        }
                    }
                }
            }
            if (!ok) {                       // gave up: the MMAs in flight read this CTA's memory
                commit(&bar.drain);
                for (uint32_t k = 0; k < kTcSpin && !mbar_try_wait(&bar.drain, 0); ++k) {
                }
            }
        }
        __syncwarp();
    } else {
        const int grp = warp >> 3, half = (warp >> 2) & 1;
        const TQ *qbase = reinterpret_cast<const TQ *>(p.q);
        // Q rows into swizzled tiles (rows behind the last: zero), a batch of loads under way at once. Without a key
        // nothing reads them, and no product stands between these stores and the rows that leave through the same memory
        const int fill = n == 0 ? 0 : (alt || nq == 1 ? 1 : 2) * kTcRows * CH;
        constexpr int QB = kSplit ? 4 : 8;
        for (int i0 = tid; i0 < fill; i0 += kTcSoftmax * QB) {
            uint4 v[QB], v2[kSplit ? QB : 1];
#pragma unroll
            for (int j = 0; j < QB; ++j) {
                const int i = i0 + kTcSoftmax * j, r = i / CH, c = i - r * CH, row = row0 + r;
                v[j] = make_uint4(0u, 0u, 0u, 0u);
                if constexpr (kSplit) v2[j] = v[j];
                if (r < nrows) {
                    const TQ *src = qbase + (long long)(q0 + row / G) * p.q_stride + (g * G + row % G) * HD + c * 8;
                    v[j] = __ldg(reinterpret_cast<const uint4 *>(src));
                    if constexpr (kSplit) v2[j] = __ldg(reinterpret_cast<const uint4 *>(src) + 1);
                }
            }
#pragma unroll
            for (int j = 0; j < QB; ++j) {
                const int i = i0 + kTcSoftmax * j, r = i / CH, c = i - r * CH;
                if (i >= fill) break;
                const uint32_t at = base + (uint32_t)(r >> 7) * L::kTile + (c >> 3) * L::kHalf + (r & 127) * 128 + (((c & 7) ^ (r & 7)) << 4);
                if constexpr (kSplit) {
                    const uint32_t x[8] = {v[j].x, v[j].y, v[j].z, v[j].w, v2[j].x, v2[j].y, v2[j].z, v2[j].w};
                    uint32_t hw[4], lw[4];
                    float top = 0.f, down, up;
#pragma unroll
                    for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(__uint_as_float(x[k])));
#pragma unroll
                    for (int k = CH / 2; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));    // a row's CH lanes
                    row_power(top, down, up);
                    if (c == 0) s_up[r] = up;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float x0 = __uint_as_float(x[2 * k]) * down, x1 = __uint_as_float(x[2 * k + 1]) * down;
                        float h0, h1;
                        hw[k] = pack2<TC>(x0, x1);
                        unpack2<TC>(hw[k], h0, h1);
                        lw[k] = pack2<TC>(x0 - h0, x1 - h1);
                    }
                    st_shared16(at, hw[0], hw[1], hw[2], hw[3]);
                    st_shared16(at + L::kTile, lw[0], lw[1], lw[2], lw[3]);
                } else {
                    st_shared16(at, v[j].x, v[j].y, v[j].z, v[j].w);
                }
            }
        }
        fence_proxy_async_smem();
        if constexpr (kSplit) asm volatile("bar.sync 9, %0;" ::"n"(kTcSoftmax) : "memory");    // s_up
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.q_full);
        if (grp < nq) {
            const int r = (alt ? 0 : grp * kTcRows) + (warp & 3) * 32 + lane, row = row0 + r;
            const bool live = r < nrows;
            const int seen = live ? own0 + row / G + 1 : 0;  // own keys this row sees: below this
            const uint32_t lanes = (uint32_t)(warp & 3) * 32u << 16;
            const uint32_t ts = tmem + lanes + 128u * grp, to = tmem + lanes + 256u + 128u * grp;
            const float up = kSplit && n > 0 ? s_up[r % (kSplit ? kTcRows : 1)] : 1.f, c = kSplit ? row_scale(p, up) : row_scale(p);
            float m = -INFINITY, l = 0.f;
            uint32_t ph = 0u;
            bool ok = true, any = false, flushed = false;
            // the two halves of a row's columns: their threads exchange a value through shared memory
            const auto swap = [&](float v) -> float {
                s_swap[grp][half][r & 127] = v;
                asm volatile("bar.sync %0, 64;" ::"r"(1 + grp * 4 + (warp & 3)) : "memory");
                return s_swap[grp][half ^ 1][r & 127];
            };
            for (int i = alt ? grp : 0; i < n; i += alt ? 2 : 1) {
                // after an expired wait the walk goes on over whatever is there: every thread keeps to its barriers
                if (ok) ok = w.wait_warp(&bar.s_full[grp], ph);
                ph ^= 1u;
                tc_fence_after();
                const int lo = ks.lo(i), lim = min(ks.hi(i), i >= own_tile0 ? seen : INT_MAX) - lo - 64 * half;
                const bool cut = __any_sync(0xffffffffu, lim < 64);
                // 32 columns at a time, read again for the exponentials: half the registers, and four warps a
                // scheduler instead of two
                const auto scores = [&](int k, uint32_t (&s)[32]) {
                    tmem_ld32_nowait(ts + 64 * half + 32 * k, s);
                    tmem_wait_ld();
                    if (cut) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (32 * k + j >= lim) s[j] = 0xff800000u;                // -inf
                    }
                };
                float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    uint32_t s[32];
                    scores(k, s);
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        mx[0] = max3(mx[0], __uint_as_float(s[j]), __uint_as_float(s[j + 1]));
                        mx[1] = max3(mx[1], __uint_as_float(s[j + 2]), __uint_as_float(s[j + 3]));
                    }
                }
                const float mine = fmaxf(mx[0], mx[1]), mt = fmaxf(mine, swap(mine));
                const bool grow = (mt - m) * c > kTcGrow<TQ, TC> || (!any && mt > m);
                const bool flush = kSplit && !alt && i > 0 && i % kTcFlush == 0;
                if (any && (flush || __any_sync(0xffffffffu, grow))) {
                    // s_full of this tile came after the products of the tile before: O is at rest
                    const float f = grow ? exp2_approx((m - mt) * c) : 1.f;
                    l *= f;
#pragma unroll 1
                    for (int k = 0; k < HD / 32; ++k) {
                        const uint32_t at = to + HD / 2 * half + 16 * k;
                        uint32_t o[16], t[16];
                        tmem_ld16_nowait(at, o);
                        if (flushed) tmem_ld16_nowait(at + 128, t);
                        tmem_wait_ld();
                        if (flush || flushed) {
#pragma unroll
                            for (int j = 0; j < 16; ++j)
                                t[j] = __float_as_uint(((flushed ? __uint_as_float(t[j]) : 0.f) + (flush ? __uint_as_float(o[j]) : 0.f)) * f);
                            tmem_st16(at + 128, t);
                        }
                        if (!flush) {                        // else the tile's products start O anew
#pragma unroll
                            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                            tmem_st16(at, o);
                        }
                    }
                    flushed |= flush;
                }
                if (grow) m = mt;
                any = true;
                const float ms = m == -INFINITY ? 0.f : m;
                // the difference costs an instruction for two columns (packed prompts 196.5 -> 199 us); a second loop
                // without it, for scores small enough, took 211
                const uint64_t c2 = f2(c, c), m2 = f2(-ms, -ms), k2 = f2(kTcBias<TQ, TC>, kTcBias<TQ, TC>);
                uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    uint32_t s[32], hi[16], lw[16];
                    scores(k, s);
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const uint64_t x = fma2(add2((uint64_t)s[2 * j] | ((uint64_t)s[2 * j + 1] << 32), m2), c2, k2);
                        const float e0 = exp2_approx(f2_lo(x)), e1 = exp2_approx(f2_hi(x));
                        sum[j & 1] = add2(sum[j & 1], f2(e0, e1));
                        hi[j] = pack2<TC>(e0, e1);
                        if constexpr (kSplit) {
                            float h0, h1;
                            unpack2<TC>(hi[j], h0, h1);
                            lw[j] = pack2<TC>(e0 - h0, e1 - h1);
                        }
                    }
                    // in place of the 32 scores: 16 columns of P, and of its lo half
                    tmem_st16(ts + 64 * half + 32 * k, hi);
                    if constexpr (kSplit) tmem_st16(ts + 64 * half + 32 * k + 16, lw);
                }
                sum[0] = add2(sum[0], sum[1]);
                l += f2_lo(sum[0]) + f2_hi(sum[0]);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar.p_full[grp]);
                // the next tile's swap writes what this one read: this tile's MMAs lie between (s_full)
            }
            // O and the row's statistics, half of the dims per thread. A warp's 32 half rows go through shared memory
            // (the tiles are done with once both groups' products are) and out as whole rows: a thread storing its
            // own row, 16 bytes of 32 rows at a time, took 4 us, a bulk copy per row 2.5
            for (int q = 0; q < nq; ++q)
                if (ok && (alt ? q < n : n > 0)) ok = w.wait_warp(&bar.o_full[q], 0);
            tc_fence_after();
            constexpr float kUnbias = 1.0f / (1 << (int)kTcBias<TQ, TC>);
            l = (l + swap(l)) * kUnbias;
            const long long rt = q0 + row / G, hh = g * G + row % G;
            const long long at = ((long long)(slot + (alt ? grp : 0)) * ba.T + rt) * p.nh + hh;
            const bool direct = pl.slots == 1;
            const float out = (!direct ? 1.f : l > 0.f ? 1.f / l : 0.f) * kUnbias;
            constexpr int HALF = HD / 2, STRIDE = HALF * 4 + 16;
            const uint32_t stage = base + (uint32_t)warp * 32 * STRIDE;
#pragma unroll
            for (int k = 0; k < HALF / 32; ++k) {
                uint32_t o[32];
                if (any && ok) {
                    tmem_ld32_nowait(to + HALF * half + 32 * k, o);
                    tmem_wait_ld();
                    if (flushed) {
                        uint32_t t[32];
                        tmem_ld32_nowait(to + 128 + HALF * half + 32 * k, t);
                        tmem_wait_ld();
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) + __uint_as_float(t[j]));
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) o[j] = 0u;
                }
#pragma unroll
                for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(!direct || l == l ? __uint_as_float(o[j]) * out : l);
                const uint32_t mine = stage + lane * STRIDE;
                if (direct && !kSplit) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t v[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] = pack2<TC>(__uint_as_float(o[8 * j + 2 * i]), __uint_as_float(o[8 * j + 2 * i + 1]));
                        st_shared16(mine + 64 * k + 16 * j, v[0], v[1], v[2], v[3]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) st_shared16(mine + 128 * k + 16 * j, o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
                }
            }
            // each lane knows where its own row goes
            uint8_t *dst = direct ? reinterpret_cast<uint8_t *>(reinterpret_cast<TQ *>(p.out) + rt * p.out_stride + hh * HD + HALF * half)
                                  : reinterpret_cast<uint8_t *>(pl.acc + at * HD + HALF * half);
            if (!live) dst = nullptr;
            __syncwarp();
            const int per = (direct ? HALF * (int)sizeof(TQ) : HALF * 4) / 16, rows = 32 / per;    // lanes a row, rows at once
#pragma unroll 4
            for (int i = 0; i < 32; i += rows) {
                const int from = i + lane / per, c16 = lane % per * 16;
                uint8_t *d = reinterpret_cast<uint8_t *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), from));
                uint4 v;
                asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                             : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(stage + from * STRIDE + c16));
                if (d) *reinterpret_cast<uint4 *>(d + c16) = v;
            }
            if (live && half == 0) {
                if (!direct) *reinterpret_cast<float2 *>(pl.ml + at * 2) = make_float2(m * up, l);
                else if (p.lse) p.lse[rt * p.nh + hh] = row_lse(m, l, c);
            }
            tc_fence_before();
        }
    }
    __syncthreads();
    if (warp == kTcMma) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
    }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled() {
    static const EncodeTiledFn fn = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &r) != cudaSuccess ||
            r != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<EncodeTiledFn>(f);
    }();
    return fn;
}

// [dims][slots][heads][pages] of one of K and V; a box is 64 dims of a page's slots (128 at most)
cudaError_t pages_map(CUtensorMap *m, const PagesView &pg, void *base, bool bf16) {
    const EncodeTiledFn enc = encode_tiled();
    if (!enc) return cudaErrorNotSupported;
    const cuuint64_t dims[4] = {(cuuint64_t)pg.hd, (cuuint64_t)pg.page_size, (cuuint64_t)pg.nkv, (cuuint64_t)pg.n_pages};
    // a dimension of one entry has no stride of its own
    const cuuint64_t any = (cuuint64_t)pg.hd * 2;
    const cuuint64_t strides[3] = {pg.page_size > 1 ? (cuuint64_t)pg.slot_stride * 2 : any,
                                   pg.nkv > 1 ? (cuuint64_t)pg.head_stride * 2 : any,
                                   pg.n_pages > 1 ? (cuuint64_t)pg.page_stride * 2 : any};
    const cuuint32_t box[4] = {64, (cuuint32_t)std::min(pg.page_size, kTcKeys), 1, 1}, one[4] = {1, 1, 1, 1};
    const CUresult r = enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, base, dims, strides, box,
                           one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <int HD, typename TQ, typename TC>
cudaError_t tc_typed(const PagesAttention &p, const PagesPlan &pl, cudaStream_t s) {
    CUtensorMap k, v;
    cudaError_t e = pages_map(&k, p.pg, p.pg.k, !std::is_same<TC, __half>::value);
    if (e == cudaSuccess) e = pages_map(&v, p.pg, p.pg.v, !std::is_same<TC, __half>::value);
    if (e == cudaSuccess) e = raise_smem(k_pages_tc<HD, TQ, TC>, TcSmem<HD>::kBytes);
    if (e != cudaSuccess) return e;
    const int items = (pl.prefix_tc ? pl.prefix_tiles * pl.prefix_splits : 0) +
                      (pl.own_tc ? p.ba.B * pl.own_tiles * (pl.whole ? 1 : pl.own_splits) : 0);
    k_pages_tc<HD, TQ, TC><<<dim3(items, p.pg.nkv), kTcThreads, TcSmem<HD>::kBytes, s>>>(k, v, p, pl);
    return cudaGetLastError();
}

}  // namespace

// Pages whose slots a TMA box takes whole and whose rows land on swizzle atoms.
bool pages_tc_fits(const PagesView &pg) {
    const bool pow2 = pg.page_size >= 8 && pg.page_size <= 4096 && (pg.page_size & (pg.page_size - 1)) == 0;
    const auto ok = [](long long s) { return s > 0 && s < (1ll << 38); };
    return pow2 && ok(pg.slot_stride) && (pg.nkv == 1 || ok(pg.head_stride)) && (pg.n_pages == 1 || ok(pg.page_stride)) &&
           encode_tiled() != nullptr;
}

cudaError_t launch_pages_tc(const PagesAttention &p, const PagesPlan &pl, cudaStream_t s) {
    const bool wide = p.pg.hd == 128;
    if (p.q_type == VT_F32)
        return wide ? tc_typed<128, float, __half>(p, pl, s) : tc_typed<64, float, __half>(p, pl, s);
    if (p.q_type == VT_F16)
        return wide ? tc_typed<128, __half, __half>(p, pl, s) : tc_typed<64, __half, __half>(p, pl, s);
    return wide ? tc_typed<128, __nv_bfloat16, __nv_bfloat16>(p, pl, s) : tc_typed<64, __nv_bfloat16, __nv_bfloat16>(p, pl, s);
}

}  // namespace sp
