// Verification of a batch's chains of drafted tokens with given random numbers (sp_accept_chains).
//
// p_i = softmax(target row i / T), q_i = softmax(draft row i / T); draft i stays while u_i q_i(x_i) <
// p_i(x_i); the next token is drawn from max(p - q, 0) of the first refused row, or from p_n. Bound by
// reading the logits once, which is k_chain_stats; what is decided is decided in fp64:
//   k_chain_stats  (row, chunk): the chunk's maximum, its first index, and the sum of exp((l - max) / T), in
//                  fp32. In fp64 this pass was bound by the exponentials (159 against 40 us for 352 rows of
//                  152,064).
//   k_chain_draw   one cluster of 8 CTAs per request. The rows' sums decide a draft when u q and p differ by more
//                  than the sums may be off (kChainSlack); otherwise the cluster sums that pair of rows again in
//                  fp64. The row that is drawn from is summed in fp64 in any case: a draw compares a running
//                  sum over the vocabulary with a given number, and an fp32 sum of 1e5 terms would move the
//                  border by more than many tokens' whole probability. An eighth of the vocabulary per CTA (the
//                  rows mostly still in L2), sums exchanged through distributed shared memory; the CTA that
//                  holds the drawn number finds its index.
// How far k_chain_stats' sum may be off, relatively: z = (l - max) / T in base 2 carries two roundings and 1 / T a
// third (3 2^-24 |z|, and terms below 2^-60 of the largest weigh nothing: 2^-16.5 at |z| = 60), the
// exponential 2^-22, the sums over a thread's 32 terms, a warp, a CTA and the chunks at most 60 2^-24: below
// 2^-16 together; u q / p takes two such sums.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>

#include "pages.cuh"

namespace sp {

namespace {

constexpr int kStatThreads = 256;
constexpr int kStatChunk = 8192;             // logits per CTA of k_chain_stats
constexpr int kStatPer = kStatChunk / kStatThreads;
constexpr int kDrawCtas = 8;                 // CTAs (a cluster) per request
constexpr int kDrawThreads = 512;
constexpr int kDrawWarps = kDrawThreads / 32;
constexpr int kBatch = 8;                    // logits a thread of k_chain_draw has under way
constexpr double kChainSlack = 1.0 / 16384;  // 2^-14: four times two sums' bound

struct ChainStat {                           // of a chunk or a row
    float sum;                               // sum of exp((l - max) / T)
    float max;                               // NaN ignored; -inf: no logit weighs anything
    int first;                               // first index of the maximum
    int pad_;
};
SP_DEVINL float chain_k2(const ChainArgs &a, int b) {        // log2(e) / T; 0: greedy
    if (!a.temperature) return 1.4426950408889634f;
    const float t = a.temperature[b];
    return t > 0.f ? 1.4426950408889634f / t : 0.f;
}
SP_DEVINL double chain_inv_t(const ChainArgs &a, int b) {    // 0: greedy
    if (!a.temperature) return 1.0;
    const float t = a.temperature[b];
    return t > 0.f ? 1.0 / (double)t : 0.0;
}
// exp((l - m) / T), approximate: 1 at the maximum (also an infinite one), 0 for NaN and -inf
SP_DEVINL float weight32(float l, float m, float k2) {
    const float e = exp2_approx((l - m) * k2);
    return l < m ? e : l == m ? 1.f : 0.f;
}
SP_DEVINL void stat_join(ChainStat &a, const ChainStat &b, float k2) {
    if (b.max == -INFINITY) return;
    if (a.max == -INFINITY) {
        a = b;
        return;
    }
    if (b.max > a.max || (b.max == a.max && b.first < a.first)) {
        a.sum = fmaf(a.sum, weight32(a.max, b.max, k2), b.sum);
        a.max = b.max;
        a.first = b.first;
    } else {
        a.sum = fmaf(b.sum, weight32(b.max, a.max, k2), a.sum);
    }
}
SP_DEVINL int chain_count(const ChainArgs &a, int b) { return a.counts ? min(max(a.counts[b], 0), a.n) : a.n; }
// row r of request b: r <= n the target's, else the drafter's r - n - 1
template <typename T>
SP_DEVINL const T *chain_row(const ChainArgs &a, int b, int r) {
    return r <= a.n ? static_cast<const T *>(a.target) + b * a.target_bs + r * a.target_ld
                    : static_cast<const T *>(a.draft) + b * a.draft_bs + (long long)(r - a.n - 1) * a.draft_ld;
}
__host__ __device__ inline int chain_rows(const ChainArgs &a) { return a.draft ? 2 * a.n + 1 : a.n + 1; }
__host__ __device__ inline int chain_chunks(int V) { return (V + kStatChunk - 1) / kStatChunk; }

template <typename T>
__global__ void __launch_bounds__(kStatThreads) k_chain_stats(ChainArgs a, ChainStat *st) {
    __shared__ ChainStat s_st[kStatThreads / 32];
    griddep_launch_dependents();
    const int chunks = chain_chunks(a.V), rows = chain_rows(a), tid = threadIdx.x;
    const int br = blockIdx.x / chunks, chunk = blockIdx.x - br * chunks, b = br / rows, r = br - b * rows;
    const int cnt = chain_count(a, b);
    if (r <= a.n ? r > cnt : r - a.n - 1 >= cnt) return;     // a row behind the request's drafts
    const float k2 = chain_k2(a, b);
    const T *row = chain_row<T>(a, b, r);
    const int lo = chunk * kStatChunk, hi = min(a.V, lo + kStatChunk);
    constexpr int VEC = 16 / sizeof(T);
    // value i of this thread is logit lo + at(i); 16-byte loads where the row allows them
    const bool wide = (reinterpret_cast<uintptr_t>(row) & 15u) == 0 && hi - lo == kStatChunk;
    const auto at = [&](int i) { return wide ? ((i / VEC) * kStatThreads + tid) * VEC + i % VEC : i * kStatThreads + tid; };
    float v[kStatPer], m = -INFINITY;
    if (wide) {
#pragma unroll
        for (int i = 0; i < kStatPer / VEC; ++i) {
            const uint4 x = __ldg(reinterpret_cast<const uint4 *>(row + lo) + i * kStatThreads + tid);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (sizeof(T) == 4) v[4 * i + j] = __uint_as_float(w[j]);
                else unpack2<T>(w[j], v[8 * i + 2 * j], v[8 * i + 2 * j + 1]);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < kStatPer; ++i) {
            const int j = lo + i * kStatThreads + tid;
            v[i] = j < hi ? to_float(row[j]) : -INFINITY;
        }
    }
#pragma unroll
    for (int i = 0; i < kStatPer; ++i) m = fmaxf(m, v[i]);
    const float wm = warp_max(m);
    // the first index of the warp's maximum
    int first = INT_MAX;
    if (m == wm) {
#pragma unroll
        for (int i = kStatPer - 1; i >= 0; --i)
            if (v[i] == wm) first = lo + at(i);
    }
    first = __reduce_min_sync(0xffffffffu, first);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kStatPer; ++i) sum += weight32(v[i], wm, k2);
    sum = warp_sum(sum);
    if ((tid & 31) == 0) s_st[tid >> 5] = ChainStat{sum, wm, first, 0};
    __syncthreads();
    if (tid == 0) {
        ChainStat x = s_st[0];
        for (int w = 1; w < kStatThreads / 32; ++w) stat_join(x, s_st[w], k2);
        st[blockIdx.x] = x;
    }
}

// ---- exponentials in 64 bits -------------------------------------------------------------------
// Table-driven (Tang 1989): z / (ln 2 / 64) = n + f, |f| <= 1/2, by adding 1.5 2^52; e^z = 2^(n >> 6) 2^((n & 63) / 64)
// e^(f ln 2 / 64), the last by its Taylor polynomial of degree 4 (relative error below 4e-14). Eleven fp64
// operations.
__constant__ double c_exp_tab[64] = {         // 2^(i / 64)
    0x1.0000000000000p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0, 0x1.0874518759bc8p+0, 0x1.0b5586cf9890fp+0,
    0x1.0e3ec32d3d1a2p+0, 0x1.11301d0125b51p+0, 0x1.1429aaea92de0p+0, 0x1.172b83c7d517bp+0, 0x1.1a35beb6fcb75p+0,
    0x1.1d4873168b9aap+0, 0x1.2063b88628cd6p+0, 0x1.2387a6e756238p+0, 0x1.26b4565e27cddp+0, 0x1.29e9df51fdee1p+0,
    0x1.2d285a6e4030bp+0, 0x1.306fe0a31b715p+0, 0x1.33c08b26416ffp+0, 0x1.371a7373aa9cbp+0, 0x1.3a7db34e59ff7p+0,
    0x1.3dea64c123422p+0, 0x1.4160a21f72e2ap+0, 0x1.44e086061892dp+0, 0x1.486a2b5c13cd0p+0, 0x1.4bfdad5362a27p+0,
    0x1.4f9b2769d2ca7p+0, 0x1.5342b569d4f82p+0, 0x1.56f4736b527dap+0, 0x1.5ab07dd485429p+0, 0x1.5e76f15ad2148p+0,
    0x1.6247eb03a5585p+0, 0x1.6623882552225p+0, 0x1.6a09e667f3bcdp+0, 0x1.6dfb23c651a2fp+0, 0x1.71f75e8ec5f74p+0,
    0x1.75feb564267c9p+0, 0x1.7a11473eb0187p+0, 0x1.7e2f336cf4e62p+0, 0x1.82589994cce13p+0, 0x1.868d99b4492edp+0,
    0x1.8ace5422aa0dbp+0, 0x1.8f1ae99157736p+0, 0x1.93737b0cdc5e5p+0, 0x1.97d829fde4e50p+0, 0x1.9c49182a3f090p+0,
    0x1.a0c667b5de565p+0, 0x1.a5503b23e255dp+0, 0x1.a9e6b5579fdbfp+0, 0x1.ae89f995ad3adp+0, 0x1.b33a2b84f15fbp+0,
    0x1.b7f76f2fb5e47p+0, 0x1.bcc1e904bc1d2p+0, 0x1.c199bdd85529cp+0, 0x1.c67f12e57d14bp+0, 0x1.cb720dcef9069p+0,
    0x1.d072d4a07897cp+0, 0x1.d5818dcfba487p+0, 0x1.da9e603db3285p+0, 0x1.dfc97337b9b5fp+0, 0x1.e502ee78b3ff6p+0,
    0x1.ea4afa2a490dap+0, 0x1.efa1bee615a27p+0, 0x1.f50765b6e4540p+0, 0x1.fa7c1819e90d8p+0};

struct Weigh {                               // exp((l - max) / T) of a row's logits
    const double *tab;                       // c_exp_tab in shared memory
    double k;                                // 64 / (T ln 2)
    float k2;                                // 1 / (T ln 2), to leave out what is 0 in 64 bits
    // without a branch, so that several are under way in a thread
    SP_DEVINL double operator()(float l, float m) const {
        const bool some = (l - m) * k2 > -1000.f;            // no for NaN, -inf and an infinite maximum
        const double y = fma((double)l, k, -((double)m * k));   // m k is rounded once for the row
        const double t = y + 0x1.8p52;
        const int n = __double2loint(t);
        const double f = y - (t - 0x1.8p52);
        double p = fma(f, 0x1.3b2ab6fba4e77p-31, 0x1.c6b08d704a0c0p-23);
        p = fma(p, f, 0x1.ebfbdff82c58fp-15);
        p = fma(p, f, 0x1.62e42fefa39efp-7);
        p = fma(p, f, 1.0);
        const double s = tab[n & 63];
        const double e = p * __hiloint2double(__double2hiint(s) + ((n >> 6) << 20), __double2loint(s));
        return some ? e : l == m ? 1.0 : 0.0;
    }
};

SP_DEVINL void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
SP_DEVINL double ld_peer(const double *p, uint32_t rank) {
    uint32_t at;
    double v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(at) : "memory");
    return v;
}

template <typename T>
__global__ void __cluster_dims__(kDrawCtas, 1, 1) __launch_bounds__(kDrawThreads) k_chain_draw(ChainArgs a, const ChainStat *st) {
    __shared__ ChainStat s_row[2 * kChainMaxDrafts + 1];
    __shared__ double s_tab[64], s_warp[2][kDrawWarps], s_ex[2][2], s_all[2][kDrawCtas];
    __shared__ int s_dec[kChainMaxDrafts], s_pick, s_last;
    const int b = blockIdx.x / kDrawCtas, rank = blockIdx.x - b * kDrawCtas;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rows = chain_rows(a), chunks = chain_chunks(a.V), cnt = chain_count(a, b);
    const double inv_t = chain_inv_t(a, b);
    const float k2 = chain_k2(a, b);
    const Weigh weigh{s_tab, inv_t * 92.33248261689365807103517958412109, k2};
    const int *tokens = a.tokens + (size_t)b * a.n;
    const double *u = a.u + (size_t)b * (a.n + 1);
    if (tid < 64) s_tab[tid] = c_exp_tab[tid];
    if (tid == 0) {
        s_pick = INT_MAX;
        s_last = -1;
    }
    griddep_wait();
    // the rows' statistics: a warp per row, lanes over the chunks
    for (int r = warp; r < rows; r += kDrawWarps) {
        ChainStat x{0.f, -INFINITY, INT_MAX, 0};
        if (r <= a.n ? r <= cnt : r - a.n - 1 < cnt) {
            const ChainStat *c = st + ((size_t)b * rows + r) * chunks;
            for (int k = lane; k < chunks; k += 32) stat_join(x, c[k], k2);
            for (int o = 16; o > 0; o >>= 1) {
                ChainStat y{__shfl_xor_sync(0xffffffffu, x.sum, o), __shfl_xor_sync(0xffffffffu, x.max, o),
                            __shfl_xor_sync(0xffffffffu, x.first, o), 0};
                stat_join(x, y, k2);
            }
        }
        if (lane == 0) s_row[r] = x;
    }
    __syncthreads();
    // thread i decides draft i: 0 refused, 1 accepted, 2 too near to say
    if (tid < cnt) {
        const int x = tokens[tid];
        const ChainStat tp = s_row[tid];
        int dec = 0;
        if (x >= 0 && x < a.V && tp.max > -INFINITY) {
            if (inv_t == 0.0) {
                dec = x == tp.first;
            } else {
                const double px = weigh(to_float(chain_row<T>(a, b, tid)[x]), tp.max) / tp.sum;
                double qx = 1.0;
                if (a.draft) {
                    const ChainStat dq = s_row[a.n + 1 + tid];
                    qx = dq.max > -INFINITY ? weigh(to_float(chain_row<T>(a, b, a.n + 1 + tid)[x]), dq.max) / dq.sum : 0.0;
                }
                const double uq = u[tid] * qx;
                dec = px == 0.0 ? 0 : fabs(uq - px) <= kChainSlack * px ? 2 : uq < px;
            }
        }
        s_dec[tid] = dec;
    }
    __syncthreads();

    // this CTA's slice of the vocabulary, a contiguous piece of it per warp
    const int slice = (a.V + kDrawCtas - 1) / kDrawCtas, piece = (slice + kDrawWarps - 1) / kDrawWarps;
    const int s_lo = min(a.V, rank * slice), s_hi = min(a.V, s_lo + slice);
    const int w_lo = min(s_hi, s_lo + warp * piece), w_hi = min(s_hi, w_lo + piece);
    int round = 0;
    // two sums over the cluster, the same bits in every thread: each warp's x, y -> the CTAs' in s_all, the
    // totals in x, y
    const auto exchange = [&](double &x, double &y) {
        for (int o = 16; o > 0; o >>= 1) {
            x += __shfl_xor_sync(0xffffffffu, x, o);
            y += __shfl_xor_sync(0xffffffffu, y, o);
        }
        __syncthreads();                                     // s_warp and s_all of the round before are read
        if (lane == 0) {
            s_warp[0][warp] = x;
            s_warp[1][warp] = y;
        }
        __syncthreads();
        if (tid < 2) {
            double sum = 0.0;
            for (int w = 0; w < kDrawWarps; ++w) sum += s_warp[tid][w];
            s_ex[round & 1][tid] = sum;                      // a peer reads it before the barrier after next
        }
        cluster_barrier();
        if (tid < 2 * kDrawCtas) s_all[tid & 1][tid >> 1] = ld_peer(&s_ex[round & 1][tid & 1], tid >> 1);
        __syncthreads();
        ++round;
        x = y = 0.0;
        for (int c = 0; c < kDrawCtas; ++c) {
            x += s_all[0][c];
            y += s_all[1][c];
        }
    };
    // the sums of target row i and, with a drafter, draft row i
    const auto pair_sums = [&](int i, bool both, double &sp, double &sq) {
        const T *pr = chain_row<T>(a, b, i), *qr = both ? chain_row<T>(a, b, a.n + 1 + i) : pr;
        const float mp = s_row[i].max, mq = both ? s_row[a.n + 1 + i].max : 0.f;
        sp = sq = 0.0;
        for (int j0 = w_lo + lane; j0 < w_hi; j0 += 32 * kBatch) {
            float x[kBatch], y[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const int j = j0 + 32 * i;
                x[i] = j < w_hi ? to_float(pr[j]) : -INFINITY;
                y[i] = both && j < w_hi ? to_float(qr[j]) : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < kBatch; ++i) sp += weigh(x[i], mp);
            if (both) {
#pragma unroll
                for (int i = 0; i < kBatch; ++i) sq += weigh(y[i], mq);
            }
        }
        exchange(sp, sq);
    };

    int acc = 0;
    double sp = 0.0, sq = 0.0;
    bool summed = false;                                     // sp, sq are those of row acc
    for (; acc < cnt; ++acc) {                               // the same walk in every thread of the cluster
        int dec = s_dec[acc];
        summed = false;
        if (dec == 2) {
            const bool both = a.draft && s_row[a.n + 1 + acc].max > -INFINITY;
            pair_sums(acc, both, sp, sq);
            summed = true;
            const int x = tokens[acc];
            const double px = weigh(to_float(chain_row<T>(a, b, acc)[x]), s_row[acc].max) / sp;
            const double qx = both ? weigh(to_float(chain_row<T>(a, b, a.n + 1 + acc)[x]), s_row[a.n + 1 + acc].max) / sq
                                   : a.draft ? 0.0 : 1.0;
            dec = u[acc] * qx < px;
        }
        if (dec == 0) break;
    }
    const ChainStat tp = s_row[acc];
    int pick = -1;
    bool write = rank == 0;                                  // of the drawn token
    if (inv_t == 0.0) {
        if (tp.max > -INFINITY) pick = tp.first;
    } else if (tp.max > -INFINITY) {
        write = false;
        // the weights: max(p - q, 0), or p (all accepted; or nothing left of p - q)
        const bool refused = acc < cnt;
        const T *pr = chain_row<T>(a, b, acc);
        const int x = refused ? tokens[acc] : -1;
        const bool both = refused && a.draft && s_row[a.n + 1 + acc].max > -INFINITY;
        const T *qr = both ? chain_row<T>(a, b, a.n + 1 + acc) : nullptr;
        const float mq = both ? s_row[a.n + 1 + acc].max : 0.f;
        // without a drafter's row the weights are p's, less the refused token: no sum to divide by
        if (both && !summed) pair_sums(acc, true, sp, sq);
        const double ip = both ? 1.0 / sp : 0.0, iq = both ? 1.0 / sq : 0.0;
        bool residual = refused && (both || !a.draft);       // a drafter's row that weighs nothing takes nothing away
        // both products rounded (no fused multiply-add): equal rows leave exactly nothing
        const auto left = [&](int j) -> double {
            if (both && residual)
                return fmax(__dmul_rn(weigh(to_float(pr[j]), tp.max), ip) - __dmul_rn(weigh(to_float(qr[j]), mq), iq), 0.0);
            return residual && j == x ? 0.0 : weigh(to_float(pr[j]), tp.max);    // p(x) - 1 is not positive
        };
        double total;
        for (;;) {
            double none = 0.0;
            total = 0.0;
            for (int j0 = w_lo + lane; j0 < w_hi; j0 += 32 * kBatch) {
                float lp[kBatch], lq[kBatch];
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    const int j = j0 + 32 * i;
                    lp[i] = j < w_hi ? to_float(pr[j]) : -INFINITY;
                    lq[i] = both && residual && j < w_hi ? to_float(qr[j]) : -INFINITY;
                }
                if (both && residual) {
#pragma unroll
                    for (int i = 0; i < kBatch; ++i)
                        total += fmax(__dmul_rn(weigh(lp[i], tp.max), ip) - __dmul_rn(weigh(lq[i], mq), iq), 0.0);
                } else {
#pragma unroll
                    for (int i = 0; i < kBatch; ++i)
                        total += weigh(residual && j0 + 32 * i == x ? -INFINITY : lp[i], tp.max);
                }
            }
            exchange(total, none);
            if (total > 0.0 || !residual) break;
            residual = false;                                // nothing left of p - q: p itself
        }
        // the first CTA, warp and index whose running sum passes `want`; where rounding lets none of them
        // pass it, the last one that weighs anything
        const double want = u[a.n] * total;
        double run = 0.0, before = 0.0;
        int owner = -1;
        for (int c = 0; c < kDrawCtas; ++c) {
            const double next = run + s_all[0][c];
            if (s_all[0][c] > 0.0) {
                owner = c;
                before = run;
                if (next > want) break;
            }
            run = next;
        }
        if (owner == rank) {
            int w_own = 0;
            double base = before;
            run = before;
            for (int w = 0; w < kDrawWarps; ++w) {
                const double next = run + s_warp[0][w];
                if (s_warp[0][w] > 0.0) {
                    w_own = w;
                    base = run;
                    if (next > want) break;
                }
                run = next;
            }
            // that warp's piece again, a few indices a thread
            const int p_lo = min(s_hi, s_lo + w_own * piece), p_hi = min(s_hi, p_lo + piece);
            const int per = (p_hi - p_lo + kDrawThreads - 1) / kDrawThreads;
            const int t_lo = min(p_hi, p_lo + tid * per), t_hi = min(p_hi, t_lo + per);
            double mine = 0.0;
            int last = -1;
            for (int j = t_lo; j < t_hi; ++j) {
                const double w = left(j);
                mine += w;
                if (w > 0.0) last = j;
            }
            double incl = mine;
            for (int o = 1; o < 32; o <<= 1) {
                const double y = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += y;
            }
            __syncthreads();                                 // s_warp is read
            if (lane == 31) s_warp[0][warp] = incl;
            __syncthreads();
            run = base;
            for (int w = 0; w < warp; ++w) run += s_warp[0][w];
            const double from_here = run + incl - mine;
            if (mine > 0.0) {
                run = from_here;
                for (int j = t_lo; j < t_hi; ++j) {
                    const double w = left(j);
                    run += w;
                    if (w > 0.0 && run > want) {
                        atomicMin(&s_pick, j);
                        break;
                    }
                }
                atomicMax(&s_last, last);
            }
            __syncthreads();
            pick = s_pick != INT_MAX ? s_pick : s_last;
            write = true;
        }
    }
    // write: rank 0 the accepted tokens and the tail, the CTA that found it the drawn one
    int *out = a.out_tokens + (size_t)b * (a.n + 1);
    if (rank == 0) {
        for (int i = tid; i <= a.n; i += kDrawThreads)
            if (i != acc) out[i] = i < acc ? tokens[i] : -1;
        if (tid == 0) a.accepted[b] = acc;
    }
    if (write && tid == 0) out[acc] = pick;
    cluster_barrier();                                       // no CTA ends while a peer reads its sums
}

template <typename T>
cudaError_t chains_typed(const ChainArgs &a, cudaStream_t s) {
    ChainStat *st = static_cast<ChainStat *>(a.ws);
    k_chain_stats<T><<<(unsigned)(a.B * chain_rows(a) * chain_chunks(a.V)), kStatThreads, 0, s>>>(a, st);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    return launch_dependent(k_chain_draw<T>, dim3(a.B * kDrawCtas), kDrawThreads, 0, s, a, st);
}

}  // namespace

size_t chains_workspace(int B, int n, int V) { return (size_t)B * (2 * n + 1) * chain_chunks(V) * sizeof(ChainStat); }

cudaError_t launch_accept_chains(const ChainArgs &a, cudaStream_t s) {
    if (a.type == VT_F32) return chains_typed<float>(a, s);
    return a.type == VT_F16 ? chains_typed<__half>(a, s) : chains_typed<__nv_bfloat16>(a, s);
}

}  // namespace sp
