// Verification of a batch's chains of drafted tokens with given random numbers (sp_accept_chains).
//
// p_i = softmax(target row i / T), q_i = softmax(draft row i / T); draft i stays while u_i q_i(x_i) <
// p_i(x_i); the next token is drawn from max(p - q, 0) of the first refused row, or from p_n. Bound by
// reading the logits once, which is k_chain_stats; what is decided is decided in fp64, on the one or two rows a
// request draws from (mostly still in L2):
//   k_chain_stats   (row, chunk): the chunk's maximum, its first index, and the sum of exp((l - max) / T), in
//                   fp32. In fp64 this pass was bound by the exponentials (159 against 41 us for 352 rows of
//                   152,064).
//   k_chain_sums    (request, piece of the vocabulary): joins the chunks and walks the chain (every piece's CTA for
//                   itself: less than a launch), then fp64 sums of the rows that are drawn from. The rows' fp32
//                   sums decide a draft when u q and p differ by more than the sums may be off (chain_slack); a
//                   draft that is nearer (one in 10,000) is summed as if refused and left to k_chain_pick. A draw
//                   compares a running sum over the vocabulary with a given number, and an fp32 sum of 1e5 terms
//                   would move the border by more than many tokens' whole probability.
//   k_chain_left    (request, piece): fp64 sums of max(p - q, 0), for requests with a refused draft and a drafter
//   k_chain_pick    a CTA per request: the piece and in it the index whose running sum passes u times the total
// For 32 requests' five drafts, 152,064 logits, each alone and cold: 37, 27, 20 and 13 us; together 77, at a floor of
// 32.7 (0.214 GB once, 6.5 TB/s). k_chain_stats runs at 5.7 TB/s; the others are short and wait for one another.
// The pieces spread the requests' fp64 work (four exponentials a token after a refusal, else one) over all SMs; a
// cluster of 8 CTAs per request for the last four took 43 us for 32 requests and 36 for 48 without a drafter, these
// 40 and 24.
// How far k_chain_stats' sum may be off, relatively and in units of 2^-24: z = (l - max) / T in base 2 carries four
// roundings (1 / T has two), so a term is off by 4 |z| ln 2, and terms below 2^-60 of the largest weigh nothing: 169 at
// |z| = 60 (the joins' exponents add up to z); the exponential 4; the sums over a thread's 64 terms and a warp 69; a join
// of two maxima's sums 5, one rounding and a factor's exponential, 3 of them in a CTA, 5 in a warp over the chunks and one
// for every 32 chunks: 282 + 5 ceil(chunks / 32) (chain_slack). u q / p takes two such sums: 2^-14.8 for 152,064 logits.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>

#include "pages.cuh"

namespace sp {

namespace {

constexpr int kStatThreads = 128;
constexpr int kStatMost = 64;                // logits per thread of k_chain_stats at most
constexpr int kPieceThreads = 256;
constexpr int kPieceMost = 4096;             // logits per CTA of k_chain_sums and k_chain_left at most
constexpr int kBatch = 8;                    // logits a thread has under way
constexpr int kPickThreads = 512;
// above what two sums may be off: 2^-14, and more from 12 million logits on
inline double chain_slack(int chunks) { return std::max(1.0 / 16384, 2.0 * (282 + 5 * ((chunks + 31) / 32)) / (1 << 24)); }

struct ChainStat {                           // of a chunk or a row
    float sum;                               // sum of exp((l - max) / T)
    float max;                               // NaN ignored; -inf: no logit weighs anything
    int first;                               // first index of the maximum
    int pad_;
};
// T, the largest finite number for an infinite one: 0 x -inf would be NaN, and 1 / T = 0 means greedy
SP_DEVINL float chain_t(const ChainArgs &a, int b) {
    const float t = a.temperature ? a.temperature[b] : 1.f;
    return t > FLT_MAX ? FLT_MAX : t;
}
SP_DEVINL float chain_k2(const ChainArgs &a, int b) {        // log2(e) / T; 0: greedy
    const float t = chain_t(a, b);
    return t > 0.f ? 1.4426950408889634f / t : 0.f;
}
SP_DEVINL double chain_inv_t(const ChainArgs &a, int b) {    // 0: greedy
    const float t = chain_t(a, b);
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
// Logits per CTA of k_chain_stats: 64 a thread, or 32 while that leaves SMs idle (32 requests' five drafts 79 ->
// 75 us with 64, one request's four 17 -> 19).
inline int chain_chunk(int rows, int V) {
    const int most = kStatMost * kStatThreads;
    return (long long)rows * ((V + most - 1) / most) < 4 * 148 ? most / 2 : most;
}

template <typename T, int PER>
__global__ void __launch_bounds__(kStatThreads) k_chain_stats(ChainArgs a, ChainStat *st) {
    constexpr int kStatPer = PER, kStatChunk = PER * kStatThreads;
    __shared__ ChainStat s_st[kStatThreads / 32];
    griddep_launch_dependents();
    const int chunks = (a.V + kStatChunk - 1) / kStatChunk, rows = chain_rows(a), tid = threadIdx.x;
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
// e^(f ln 2 / 64), the last by its Taylor polynomial of degree 4 (relative error below 4e-14). Twelve fp64
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
        // (l - m) k, with what the rounding of m k left off taken back (by the row): 0 at the maximum whatever T and the
        // logits' size, where at T = 1e-15, or logits of 1e20, that rest alone is as large as the exponent may be. The
        // difference first takes one operation less and 8 more registers: 54.5 against 52.4 us for 48 requests
        const double mk = (double)m * k, y = fma((double)l, k, -mk) - fma((double)m, k, -mk);
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

// ---- the draw ----------------------------------------------------------------------------------
enum ChainMode : int { CM_DONE = 0, CM_P = 1, CM_P_LESS = 2, CM_BOTH = 3, CM_NEAR = 4, CM_SLOW = 5 };
struct ChainPlan {                           // of a request, by chain_decide
    int mode;                                // weights: none (the token is written), p, p without the refused token,
                                             // max(p - q, 0); draft acc is too near to say; or two are (the slow walk)
    int acc;                                 // accepted drafts: the row that is drawn from
    float mp, mq;                            // the rows' maxima
};
struct ChainScratch {
    ChainStat *st;                           // [B][rows][chunks]
    ChainPlan *plan;                         // [B][2]: the plan; where a draft is too near, the one if it is accepted
    double *sp, *sq, *left;                  // [B][pieces]
    int piece, pieces;                       // logits of a piece, pieces of a row
    int chunk, chunks;                       // likewise of the statistics
    double slack;                            // how near u q and p leave a draft undecided, relative to p
};
// Pieces of 4,096 logits, or of half while they leave SMs idle: for one request's four drafts 18 against 21 us
// (a quarter: 20), for 32 requests 88 against 81.
inline int chain_piece(int B, int V) {
    return (long long)B * ((V + kPieceMost - 1) / kPieceMost) < 2 * 148 ? kPieceMost / 2 : kPieceMost;
}

SP_DEVINL Weigh chain_weigh_of(const ChainArgs &a, int b, const double *tab) {
    return Weigh{tab, chain_inv_t(a, b) * 92.33248261689365807103517958412109, chain_k2(a, b)};
}
SP_DEVINL Weigh chain_weigh(const ChainArgs &a, int b, double *tab) {
    if (threadIdx.x < 64) tab[threadIdx.x] = c_exp_tab[threadIdx.x];
    return chain_weigh_of(a, b, tab);
}
// sums of a CTA, the same bits in every thread
template <int THREADS>
SP_DEVINL void cta_sums(double &x, double &y, double (*s_sum)[THREADS / 32]) {
    for (int o = 16; o > 0; o >>= 1) {
        x += __shfl_xor_sync(0xffffffffu, x, o);
        y += __shfl_xor_sync(0xffffffffu, y, o);
    }
    __syncthreads();                                         // s_sum of the time before is read
    if ((threadIdx.x & 31) == 0) {
        s_sum[0][threadIdx.x >> 5] = x;
        s_sum[1][threadIdx.x >> 5] = y;
    }
    __syncthreads();
    x = y = 0.0;
    for (int w = 0; w < THREADS / 32; ++w) {
        x += s_sum[0][w];
        y += s_sum[1][w];
    }
}

struct DecideShared {
    ChainStat row[2 * kChainMaxDrafts + 1];
    int dec[kChainMaxDrafts];
};
// The walk along request b's chain, by a whole CTA; `write`: the plan and every token but the drawn one as well.
template <typename T>
SP_DEVINL ChainPlan chain_decide(const ChainArgs &a, const ChainScratch &sc, int b, const Weigh &weigh, DecideShared &sh,
                                 bool write) {
    ChainStat *s_row = sh.row;
    int *s_dec = sh.dec;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rows = chain_rows(a), chunks = sc.chunks, cnt = chain_count(a, b);
    const double inv_t = chain_inv_t(a, b);
    const float k2 = chain_k2(a, b);
    const int *tokens = a.tokens + (size_t)b * a.n;
    // thread i decides draft i: its token, and the token's logits, do not wait for the statistics
    int x = -1;
    float lp = -INFINITY, lq = -INFINITY;
    double u = 0.0;
    if (tid < cnt) {
        x = tokens[tid];
        u = a.u[(size_t)b * (a.n + 1) + tid];
        if (x >= 0 && x < a.V) {
            lp = to_float(chain_row<T>(a, b, tid)[x]);
            if (a.draft) lq = to_float(chain_row<T>(a, b, a.n + 1 + tid)[x]);
        }
    }
    griddep_wait();
    // the rows' statistics: a warp per row, lanes over the chunks
    for (int r = warp; r < rows; r += kPieceThreads / 32) {
        ChainStat s{0.f, -INFINITY, INT_MAX, 0};
        if (r <= a.n ? r <= cnt : r - a.n - 1 < cnt) {
            const ChainStat *c = sc.st + ((size_t)b * rows + r) * chunks;
            for (int k = lane; k < chunks; k += 32) stat_join(s, c[k], k2);
            for (int o = 16; o > 0; o >>= 1) {
                ChainStat y{__shfl_xor_sync(0xffffffffu, s.sum, o), __shfl_xor_sync(0xffffffffu, s.max, o),
                            __shfl_xor_sync(0xffffffffu, s.first, o), 0};
                stat_join(s, y, k2);
            }
        }
        if (lane == 0) s_row[r] = s;
    }
    __syncthreads();
    if (tid < cnt) {                                         // 0 refused, 1 accepted, 2 too near to say
        const ChainStat tp = s_row[tid];
        int dec = 0;
        if (x >= 0 && x < a.V && tp.max > -INFINITY) {
            if (inv_t == 0.0) {
                dec = x == tp.first;
            } else {
                const double px = weigh(lp, tp.max) / tp.sum;
                double qx = 1.0;
                if (a.draft) {
                    const ChainStat dq = s_row[a.n + 1 + tid];
                    qx = dq.max > -INFINITY ? weigh(lq, dq.max) / dq.sum : 0.0;
                }
                const double uq = u * qx;
                dec = px == 0.0 ? 0 : fabs(uq - px) <= sc.slack * px ? 2 : uq < px;
            }
        }
        s_dec[tid] = dec;
    }
    __syncthreads();
    int pick = -1;
    const auto walk = [&](int acc) {                         // on from draft acc
        while (acc < cnt && s_dec[acc] == 1) ++acc;
        const bool refused = acc < cnt;
        ChainPlan plan{CM_DONE, acc, s_row[acc].max, refused && a.draft ? s_row[a.n + 1 + acc].max : -INFINITY};
        pick = -1;
        if (refused && s_dec[acc] == 2) plan.mode = CM_NEAR;
        else if (plan.mp == -INFINITY) pick = -1;
        else if (inv_t == 0.0) pick = s_row[acc].first;
        else if (!refused || (a.draft && plan.mq == -INFINITY)) plan.mode = CM_P;    // a drafter's empty row takes nothing away
        else plan.mode = a.draft ? CM_BOTH : CM_P_LESS;
        return plan;
    };
    ChainPlan plan = walk(0);
    if (plan.mode == CM_NEAR) {
        const ChainPlan other = walk(plan.acc + 1);
        if (other.mode == CM_NEAR) plan.mode = CM_SLOW;
        if (write && tid == 0) sc.plan[2 * b + 1] = other;
    }
    if (write && tid == 0) sc.plan[2 * b] = plan;
    if (write && plan.mode < CM_NEAR) {
        int *out = a.out_tokens + (size_t)b * (a.n + 1);
        for (int i = tid; i <= a.n; i += kPieceThreads)
            if (i != plan.acc) out[i] = i < plan.acc ? tokens[i] : -1;
            else if (plan.mode == CM_DONE) out[i] = pick;
        if (tid == 0) a.accepted[b] = plan.acc;
    }
    return plan;
}

// f(index, logits) of a piece [lo, hi) of row pr and, if given, qr, by THREADS threads
template <typename T, int THREADS, typename F>
SP_DEVINL void walk_piece(const T *pr, const T *qr, int lo, int hi, F f) {
    for (int j0 = lo + threadIdx.x % THREADS; j0 < hi; j0 += THREADS * kBatch) {
        float x[kBatch], y[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int j = j0 + THREADS * i;
            x[i] = j < hi ? to_float(pr[j]) : -INFINITY;
            y[i] = qr && j < hi ? to_float(qr[j]) : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) f(j0 + THREADS * i, x[i], y[i]);
    }
}
// max(p - q, 0) of a token; both products rounded (no fused multiply-add): equal rows leave exactly nothing
SP_DEVINL double left_of(double ep, double ip, double eq, double iq) {
    return fmax(__dmul_rn(ep, ip) - __dmul_rn(eq, iq), 0.0);
}

template <typename T>
__global__ void __launch_bounds__(kPieceThreads) k_chain_sums(ChainArgs a, ChainScratch sc) {
    __shared__ double s_tab[64], s_sum[2][kPieceThreads / 32];
    __shared__ DecideShared s_decide;
    griddep_launch_dependents();
    const int pieces = sc.pieces, b = blockIdx.x / pieces, k = blockIdx.x - b * pieces;
    const Weigh weigh = chain_weigh(a, b, s_tab);
    __syncthreads();
    ChainPlan plan = chain_decide<T>(a, sc, b, weigh, s_decide, k == 0);
    if (plan.mode == CM_DONE || plan.mode == CM_SLOW) return;
    if (plan.mode == CM_NEAR) plan.mode = a.draft ? CM_BOTH : CM_P_LESS;     // as if it were refused
    const int lo = k * sc.piece, hi = min(a.V, lo + sc.piece);
    const T *pr = chain_row<T>(a, b, plan.acc);
    double sp = 0.0, sq = 0.0;
    if (plan.mode == CM_BOTH) {
        walk_piece<T, kPieceThreads>(pr, chain_row<T>(a, b, a.n + 1 + plan.acc), lo, hi, [&](int, float x, float y) {
            sp += weigh(x, plan.mp);
            sq += weigh(y, plan.mq);
        });
    } else {
        const int out = plan.mode == CM_P_LESS ? a.tokens[(size_t)b * a.n + plan.acc] : -1;    // p(x) - 1 is not positive
        walk_piece<T, kPieceThreads>(pr, (const T *)nullptr, lo, hi, [&](int j, float x, float) {
            sp += weigh(j == out ? -INFINITY : x, plan.mp);
        });
    }
    cta_sums<kPieceThreads>(sp, sq, s_sum);
    if (threadIdx.x == 0) {
        sc.sp[blockIdx.x] = sp;
        sc.sq[blockIdx.x] = sq;
    }
}

// a request's totals of two piece arrays: the same tree, and so the same bits, in every warp of every kernel
SP_DEVINL void piece_totals(const double *x, const double *y, int pieces, double &sx, double &sy) {
    sx = sy = 0.0;
    for (int k = threadIdx.x & 31; k < pieces; k += 32) {
        sx += x[k];
        sy += y[k];
    }
    for (int o = 16; o > 0; o >>= 1) {
        sx += __shfl_xor_sync(0xffffffffu, sx, o);
        sy += __shfl_xor_sync(0xffffffffu, sy, o);
    }
}

template <typename T>
__global__ void __launch_bounds__(kPieceThreads) k_chain_left(ChainArgs a, ChainScratch sc) {
    __shared__ double s_tab[64], s_sum[2][kPieceThreads / 32];
    griddep_launch_dependents();
    const int pieces = sc.pieces, b = blockIdx.x / pieces, k = blockIdx.x - b * pieces;
    const Weigh weigh = chain_weigh(a, b, s_tab);
    __syncthreads();
    griddep_wait();
    const ChainPlan plan = sc.plan[2 * b];
    if (plan.mode != CM_BOTH && plan.mode != CM_NEAR) return;
    double sp, sq;
    piece_totals(sc.sp + (size_t)b * pieces, sc.sq + (size_t)b * pieces, pieces, sp, sq);
    const double ip = 1.0 / sp, iq = 1.0 / sq;
    const int lo = k * sc.piece, hi = min(a.V, lo + sc.piece);
    double sum = 0.0, none = 0.0;
    walk_piece<T, kPieceThreads>(chain_row<T>(a, b, plan.acc), chain_row<T>(a, b, a.n + 1 + plan.acc), lo, hi,
                                 [&](int, float x, float y) { sum += left_of(weigh(x, plan.mp), ip, weigh(y, plan.mq), iq); });
    cta_sums<kPieceThreads>(sum, none, s_sum);
    if (threadIdx.x == 0) sc.left[blockIdx.x] = sum;
}

// A request with a draft that is too near to say, by k_chain_pick's CTA: that draft, the tokens and the sums of the rows
// that are drawn from. Not inlined: one request in some hundreds comes here (3 to 70 us more), and its code in line cost every
// call 3 us.
template <typename T>
__device__ __noinline__ ChainPlan settle_near(const ChainArgs &a, const ChainScratch &sc, int b, const double *tab,
                                              double (*s_sum)[kPickThreads / 32]) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, pieces = sc.pieces;
    const Weigh weigh = chain_weigh_of(a, b, tab);
    const double *u = a.u + (size_t)b * (a.n + 1);
    const int *tokens = a.tokens + (size_t)b * a.n;
    double *sp = sc.sp + (size_t)b * pieces, *sq = sc.sq + (size_t)b * pieces, *left = sc.left + (size_t)b * pieces;
    ChainPlan plan = sc.plan[2 * b];
    const auto maximum = [&](const T *row) {                 // NaN ignored, the same in every thread
        float m = -INFINITY;
        for (int j = tid; j < a.V; j += kPickThreads) m = fmaxf(m, to_float(row[j]));
        double d = warp_max(m);
        __syncthreads();
        if (lane == 0) s_sum[0][warp] = d;
        __syncthreads();
        d = s_sum[0][0];
        for (int w = 1; w < kPickThreads / 32; ++w) d = fmax(d, s_sum[0][w]);
        return (float)d;
    };
    // the pieces' sums by this CTA alone, a warp a piece: of p and q into sp and sq, or of max(p - q, 0) into left
    const auto sums_here = [&](const T *pr, const T *qr, bool residual, double ip, double iq, double &tx, double &ty) {
        for (int k = warp; k < pieces; k += kPickThreads / 32) {
            double x = 0.0, y = 0.0;
            walk_piece<T, 32>(pr, qr, k * sc.piece, min(a.V, (k + 1) * sc.piece), [&](int, float lp, float lq) {
                const double ep = weigh(lp, plan.mp), eq = weigh(lq, plan.mq);
                if (residual) {
                    x += left_of(ep, ip, eq, iq);
                } else {
                    x += ep;
                    y += eq;
                }
            });
            for (int o = 16; o > 0; o >>= 1) {
                x += __shfl_xor_sync(0xffffffffu, x, o);
                y += __shfl_xor_sync(0xffffffffu, y, o);
            }
            if (lane == 0) {
                (residual ? left : sp)[k] = x;
                if (!residual) sq[k] = y;
            }
        }
        __syncthreads();
        piece_totals(residual ? left : sp, residual ? left : sq, pieces, tx, ty);
        __syncthreads();                                     // read before the next sums
    };
    // what chain_decide left open
    const auto write = [&] {
        int *out = a.out_tokens + (size_t)b * (a.n + 1);
        for (int i = tid; i <= a.n; i += kPickThreads) out[i] = i < plan.acc ? tokens[i] : -1;
        if (tid == 0) a.accepted[b] = plan.acc;
        __syncthreads();                                     // the drawn token comes on top
    };
    const auto take_out = [&](const T *pr, int x) {          // the refused token out of its piece
        if (x < 0 || x >= a.V) return;
        const int k = x / sc.piece;
        double y = 0.0, none = 0.0;
        walk_piece<T, kPickThreads>(pr, (const T *)nullptr, k * sc.piece, min(a.V, (k + 1) * sc.piece),
                                    [&](int j, float l, float) { y += weigh(j == x ? -INFINITY : l, plan.mp); });
        cta_sums<kPickThreads>(y, none, s_sum);
        if (tid == 0) sp[k] = y;
        __syncthreads();
    };
    if (plan.mode == CM_NEAR) {
        // the near draft in 64 bits, by the sums that its refusal needs (without a drafter: of p without it)
        double tp, tq, qx = 1.0;
        piece_totals(sp, sq, pieces, tp, tq);
        const int x = tokens[plan.acc];
        const double wp = weigh(to_float(chain_row<T>(a, b, plan.acc)[x]), plan.mp);
        if (a.draft) qx = weigh(to_float(chain_row<T>(a, b, a.n + 1 + plan.acc)[x]), plan.mq) / tq;
        else tp += wp;
        const bool accepted = u[plan.acc] * qx < wp / tp;
        if (accepted) plan = sc.plan[2 * b + 1];
        else plan.mode = a.draft ? CM_BOTH : CM_P_LESS;
        write();
        if (plan.mode == CM_DONE) return plan;
        if (accepted) {                                      // the sums of the rows behind it
            const T *pr = chain_row<T>(a, b, plan.acc), *qr = plan.mode == CM_BOTH ? chain_row<T>(a, b, a.n + 1 + plan.acc) : nullptr;
            sums_here(pr, qr, false, 0.0, 0.0, tp, tq);
            if (plan.mode == CM_P_LESS) take_out(pr, tokens[plan.acc]);
            double none;
            if (qr) sums_here(pr, qr, true, 1.0 / tp, 1.0 / tq, qx, none);
        }
    }
    if (plan.mode == CM_SLOW) {
        // the walk on from the draft that was too near, every decision from fp64 sums
        const int cnt = chain_count(a, b);
        double tp = 0.0, tq = 0.0;
        for (;; ++plan.acc) {
            const bool last = plan.acc >= cnt;
            const T *pr = chain_row<T>(a, b, plan.acc), *qr = !last && a.draft ? chain_row<T>(a, b, a.n + 1 + plan.acc) : nullptr;
            plan.mp = maximum(pr);
            plan.mq = qr ? maximum(qr) : -INFINITY;
            plan.mode = CM_DONE;
            if (plan.mp == -INFINITY) break;
            sums_here(pr, qr, false, 0.0, 0.0, tp, tq);
            plan.mode = CM_P;
            if (last) break;
            const int x = tokens[plan.acc];
            const bool in = x >= 0 && x < a.V;
            const double px = in ? weigh(to_float(pr[x]), plan.mp) / tp : 0.0;
            const double qx = !a.draft ? 1.0 : plan.mq > -INFINITY && in ? weigh(to_float(qr[x]), plan.mq) / tq : 0.0;
            if (in && u[plan.acc] * qx < px) continue;
            if (a.draft && plan.mq > -INFINITY) {
                plan.mode = CM_BOTH;
                double none;
                sums_here(pr, qr, true, 1.0 / tp, 1.0 / tq, tq, none);
            } else if (!a.draft) {
                plan.mode = CM_P_LESS;
                take_out(pr, x);
            }
            break;
        }
        write();
        if (plan.mode == CM_DONE) return plan;
    }
    return plan;
}

template <typename T>
__global__ void __launch_bounds__(kPickThreads, 1) k_chain_pick(const __grid_constant__ ChainArgs a, const __grid_constant__ ChainScratch sc) {
    __shared__ double s_tab[64], s_sum[2][kPickThreads / 32];
    __shared__ int s_pick, s_last;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int pieces = sc.pieces;
    const Weigh weigh = chain_weigh(a, b, s_tab);
    const double *u = a.u + (size_t)b * (a.n + 1);
    const int *tokens = a.tokens + (size_t)b * a.n;
    if (tid == 0) {
        s_pick = INT_MAX;
        s_last = -1;
    }
    __syncthreads();
    griddep_wait();
    ChainPlan plan = sc.plan[2 * b];
    if (plan.mode == CM_DONE) return;
    double *sp = sc.sp + (size_t)b * pieces, *sq = sc.sq + (size_t)b * pieces, *left = sc.left + (size_t)b * pieces;
    if (plan.mode >= CM_NEAR) {
        plan = settle_near<T>(a, sc, b, s_tab, s_sum);
        if (plan.mode == CM_DONE) return;
    }
    const T *pr = chain_row<T>(a, b, plan.acc), *qr = plan.mode == CM_BOTH ? chain_row<T>(a, b, a.n + 1 + plan.acc) : nullptr;
    double tp, tq, total, ip = 0.0, iq = 0.0;
    piece_totals(sp, sq, pieces, tp, tq);
    const double *weights = sp;
    total = tp;
    int without = plan.mode == CM_P_LESS ? tokens[plan.acc] : -1;
    if (plan.mode == CM_BOTH) {
        double none;
        piece_totals(left, left, pieces, total, none);
        if (total > 0.0) {
            weights = left;
            ip = 1.0 / tp;
            iq = 1.0 / tq;
        } else {                                             // nothing left of p - q: p itself
            qr = nullptr;
            total = tp;
        }
    } else if (plan.mode == CM_P_LESS && !(total > 0.0)) {   // p is 1 at the refused token
        if (tid == 0) a.out_tokens[(size_t)b * (a.n + 1) + plan.acc] = without;
        return;
    }
    // the first piece and index whose running sum passes `want`; where rounding lets none of them pass it, the
    // last one that weighs anything
    const double want = u[a.n] * total;
    double run = 0.0, base = 0.0;
    int own = 0;
    for (int k0 = 0; k0 < pieces; k0 += 32) {                // 32 pieces at a time, every warp alike
        const double w = k0 + lane < pieces ? weights[k0 + lane] : 0.0;
        double incl = w;
        for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        const unsigned some = __ballot_sync(0xffffffffu, w > 0.0);
        const unsigned over = __ballot_sync(0xffffffffu, w > 0.0 && run + incl > want);
        if (some) {
            const int at = over ? __ffs(over) - 1 : 31 - __clz(some);
            own = k0 + at;
            base = run + __shfl_sync(0xffffffffu, incl - w, at);
            if (over) break;
        }
        run += __shfl_sync(0xffffffffu, incl, 31);
    }
    const int lo = own * sc.piece, hi = min(a.V, lo + sc.piece), per = sc.piece / kPickThreads;
    constexpr int PER = kPieceMost / kPickThreads;           // consecutive indices of a thread, `per` of them in use
    double w[PER], mine = 0.0;
    int last = -1;
    float lp[PER], lq[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int j = i < per ? lo + tid * per + i : hi;
        lp[i] = j < hi && j != without ? to_float(pr[j]) : -INFINITY;
        lq[i] = qr && j < hi ? to_float(qr[j]) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const double ep = weigh(lp[i], plan.mp);
        w[i] = qr ? left_of(ep, ip, weigh(lq[i], plan.mq), iq) : ep;
        mine += w[i];
        if (w[i] > 0.0) last = lo + tid * per + i;
    }
    double incl = mine;
    for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 31) s_sum[0][warp] = incl;
    __syncthreads();
    run = base;
    for (int k = 0; k < warp; ++k) run += s_sum[0][k];
    run += incl - mine;
    bool found = false;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        run += w[i];
        if (!found && w[i] > 0.0 && run > want) {
            found = true;
            atomicMin(&s_pick, lo + tid * per + i);
        }
    }
    if (last >= 0) atomicMax(&s_last, last);
    __syncthreads();
    if (tid == 0) a.out_tokens[(size_t)b * (a.n + 1) + plan.acc] = s_pick != INT_MAX ? s_pick : s_last;
}

size_t up16(size_t v) { return (v + 15) / 16 * 16; }
ChainScratch chain_scratch(const ChainArgs &a, void *base) {
    uint8_t *p = static_cast<uint8_t *>(base);
    const auto take = [&](size_t bytes) { uint8_t *q = p; p += up16(bytes); return q; };
    ChainScratch sc{};
    sc.chunk = chain_chunk(a.B * (2 * a.n + 1), a.V);
    sc.chunks = (a.V + sc.chunk - 1) / sc.chunk;
    sc.slack = chain_slack(sc.chunks);
    sc.piece = chain_piece(a.B, a.V);
    sc.pieces = (a.V + sc.piece - 1) / sc.piece;
    const size_t pieces = (size_t)a.B * sc.pieces * sizeof(double);
    sc.st = reinterpret_cast<ChainStat *>(take((size_t)a.B * (2 * a.n + 1) * sc.chunks * sizeof(ChainStat)));
    sc.plan = reinterpret_cast<ChainPlan *>(take((size_t)a.B * 2 * sizeof(ChainPlan)));
    sc.sp = reinterpret_cast<double *>(take(pieces));
    sc.sq = reinterpret_cast<double *>(take(pieces));
    sc.left = reinterpret_cast<double *>(take(pieces));
    return sc;
}

template <typename T>
cudaError_t chains_typed(const ChainArgs &a, cudaStream_t s) {
    const ChainScratch sc = chain_scratch(a, a.ws);
    const unsigned stats = (unsigned)(a.B * chain_rows(a) * sc.chunks);
    if (sc.chunk == kStatMost * kStatThreads)
        k_chain_stats<T, kStatMost><<<stats, kStatThreads, 0, s>>>(a, sc.st);
    else
        k_chain_stats<T, kStatMost / 2><<<stats, kStatThreads, 0, s>>>(a, sc.st);
    cudaError_t e = cudaGetLastError();
    const dim3 pieces((unsigned)(a.B * sc.pieces));
    if (e == cudaSuccess) e = launch_dependent(k_chain_sums<T>, pieces, kPieceThreads, 0, s, a, sc);
    if (e == cudaSuccess && a.draft) e = launch_dependent(k_chain_left<T>, pieces, kPieceThreads, 0, s, a, sc);
    if (e == cudaSuccess) e = launch_dependent(k_chain_pick<T>, dim3(a.B), kPickThreads, 0, s, a, sc);
    return e;
}

}  // namespace

size_t chains_workspace(int B, int n, int V) {
    ChainArgs a{};
    a.B = B;
    a.n = n;
    a.V = V;
    const ChainScratch sc = chain_scratch(a, nullptr);
    return reinterpret_cast<size_t>(sc.left) + up16((size_t)B * sc.pieces * sizeof(double));
}

cudaError_t launch_accept_chains(const ChainArgs &a, cudaStream_t s) {
    if (a.type == VT_F32) return chains_typed<float>(a, s);
    return a.type == VT_F16 ? chains_typed<__half>(a, s) : chains_typed<__nv_bfloat16>(a, s);
}

}  // namespace sp
