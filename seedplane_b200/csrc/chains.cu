// Verification of a batch's chains of drafted tokens with given random numbers (sp_accept_chains).
//
// p_i = softmax(target row i / T), q_i = softmax(draft row i / T); draft i stays while u_i q_i(x_i) <
// p_i(x_i); the next token is drawn from max(p - q, 0) of the first refused row, or from p_n. Every
// probability and sum is fp64: a draw compares a running sum over the vocabulary with a given number,
// and fp32 sums of 1e5 terms would move the border by more than many tokens' whole probability.
// Bound by reading the logits once.
//   k_chain_stats  (chunk, row): a chunk's maximum, its first index, and sum of exp((l - max) / T)
//   k_chain_draw   one cluster of 8 CTAs per request: joins the chunks, walks the chain, then sums the
//                  weights of the row it draws from (an eighth of the vocabulary per CTA, the rows
//                  mostly still in L2), exchanges the sums through distributed shared memory, and the CTA
//                  that holds the drawn number finds its index.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>

#include "pages.cuh"

namespace sp {

namespace {

constexpr int kStatThreads = 256;
constexpr int kStatChunk = 8192;             // logits per CTA of k_chain_stats
constexpr int kDrawCtas = 8;                 // CTAs (a cluster) per request
constexpr int kDrawThreads = 512;
constexpr int kDrawWarps = kDrawThreads / 32;

struct ChainStat {                           // of a chunk or a row
    double sum;                              // sum of exp((l - max) / T)
    float max;                               // NaN ignored; -inf: no logit weighs anything
    int first;                               // first index of the maximum
};
SP_DEVINL double weight(float l, float m, double inv_t) {
    if (!(l <= m) || l == -INFINITY) return 0.0;             // NaN weighs nothing
    return l == m ? 1.0 : exp(((double)l - (double)m) * inv_t);
}
SP_DEVINL void stat_join(ChainStat &a, const ChainStat &b, double inv_t) {
    if (b.max == -INFINITY) return;
    if (a.max == -INFINITY) {
        a = b;
        return;
    }
    if (b.max > a.max || (b.max == a.max && b.first < a.first)) {
        a.sum = fma(a.sum, weight(a.max, b.max, inv_t), b.sum);
        a.max = b.max;
        a.first = b.first;
    } else {
        a.sum = fma(b.sum, weight(b.max, a.max, inv_t), a.sum);
    }
}
SP_DEVINL double chain_inv_t(const ChainArgs &a, int b) {    // 0: greedy
    if (!a.temperature) return 1.0;
    const float t = a.temperature[b];
    return t > 0.f ? 1.0 / (double)t : 0.0;
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
    const int chunks = chain_chunks(a.V), rows = chain_rows(a);
    const int br = blockIdx.x / chunks, chunk = blockIdx.x - br * chunks, b = br / rows, r = br - b * rows;
    const int cnt = chain_count(a, b);
    if (r <= a.n ? r > cnt : r - a.n - 1 >= cnt) return;     // a row behind the request's drafts
    const double inv_t = chain_inv_t(a, b);
    const T *row = chain_row<T>(a, b, r);
    const int lo = chunk * kStatChunk, hi = min(a.V, lo + kStatChunk);
    constexpr int PER = kStatChunk / kStatThreads;
    float v[PER], m = -INFINITY;
    int first = INT_MAX;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int j = lo + i * kStatThreads + threadIdx.x;
        v[i] = j < hi ? to_float(row[j]) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (v[i] > m) {
            m = v[i];
            first = lo + i * kStatThreads + threadIdx.x;
        }
    }
    ChainStat x{0.0, m, first};
    for (int o = 16; o > 0; o >>= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, x.max, o);
        const int of = __shfl_xor_sync(0xffffffffu, x.first, o);
        if (om > x.max || (om == x.max && of < x.first)) {
            x.max = om;
            x.first = of;
        }
    }
    if (inv_t > 0.0) {
#pragma unroll
        for (int i = 0; i < PER; ++i) x.sum += weight(v[i], x.max, inv_t);
        for (int o = 16; o > 0; o >>= 1) x.sum += __shfl_xor_sync(0xffffffffu, x.sum, o);
    }
    if ((threadIdx.x & 31) == 0) s_st[threadIdx.x >> 5] = x;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kStatThreads / 32; ++w) stat_join(x, s_st[w], inv_t);
        st[blockIdx.x] = x;
    }
}

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
    __shared__ double s_warp[kDrawWarps], s_mine[2];
    __shared__ int s_acc, s_pick;
    const int b = blockIdx.x / kDrawCtas, rank = blockIdx.x - b * kDrawCtas;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rows = chain_rows(a), chunks = chain_chunks(a.V), cnt = chain_count(a, b);
    const double inv_t = chain_inv_t(a, b);
    // the rows' statistics: a warp per row, lanes over the chunks
    for (int r = warp; r < rows; r += kDrawWarps) {
        ChainStat x{0.0, -INFINITY, INT_MAX};
        if (r <= a.n ? r <= cnt : r - a.n - 1 < cnt) {
            const ChainStat *c = st + ((size_t)b * rows + r) * chunks;
            for (int k = lane; k < chunks; k += 32) stat_join(x, c[k], inv_t);
            for (int o = 16; o > 0; o >>= 1) {
                ChainStat y;
                y.sum = __shfl_xor_sync(0xffffffffu, x.sum, o);
                y.max = __shfl_xor_sync(0xffffffffu, x.max, o);
                y.first = __shfl_xor_sync(0xffffffffu, x.first, o);
                // the same order on both sides: the sums agree bit for bit in every lane
                ChainStat lo = (lane & o) ? y : x, hi = (lane & o) ? x : y;
                stat_join(lo, hi, inv_t);
                x = lo;
            }
        }
        if (lane == 0) s_row[r] = x;
    }
    if (tid == 0) {
        s_acc = cnt;
        s_pick = -1;
    }
    __syncthreads();
    // which drafts pass: thread i decides draft i
    if (tid < cnt) {
        const int x = a.tokens[(size_t)b * a.n + tid];
        bool ok = false;
        if (x >= 0 && x < a.V) {
            const ChainStat &tp = s_row[tid];
            if (inv_t == 0.0) {
                ok = tp.max > -INFINITY && x == tp.first;
            } else {
                const double px = weight(to_float(chain_row<T>(a, b, tid)[x]), tp.max, inv_t) / tp.sum;
                double qx = 1.0;
                if (a.draft) {
                    const ChainStat &dq = s_row[a.n + 1 + tid];
                    qx = dq.max > -INFINITY ? weight(to_float(chain_row<T>(a, b, a.n + 1 + tid)[x]), dq.max, inv_t) / dq.sum : 0.0;
                }
                ok = tp.max > -INFINITY && a.u[(size_t)b * (a.n + 1) + tid] * qx < px;
            }
        }
        if (!ok) atomicMin(&s_acc, tid);
    }
    __syncthreads();
    const int acc = s_acc;
    const ChainStat tp = s_row[acc];
    int pick = -1;
    bool write = rank == 0;                                  // of the drawn token
    if (inv_t == 0.0) {
        if (tp.max > -INFINITY) pick = tp.first;
    } else if (tp.max > -INFINITY) {
        write = false;
        // the weights: max(p - q, 0), or p (all accepted; or nothing left of p - q)
        const T *prow = chain_row<T>(a, b, acc);
        const bool refused = acc < cnt;
        const int x = refused ? a.tokens[(size_t)b * a.n + acc] : -1;
        const T *qrow = refused && a.draft ? chain_row<T>(a, b, a.n + 1 + acc) : nullptr;
        const ChainStat dq = qrow ? s_row[a.n + 1 + acc] : ChainStat{1.0, 0.f, 0};
        const double ip = 1.0 / tp.sum, iq = dq.max > -INFINITY ? 1.0 / dq.sum : 0.0;
        bool residual = refused;
        const auto left = [&](int j) -> double {
            double w = weight(to_float(prow[j]), tp.max, inv_t) * ip;
            if (!residual) return w;
            if (qrow) return fmax(w - weight(to_float(qrow[j]), dq.max, inv_t) * iq, 0.0);
            return j == x ? fmax(w - 1.0, 0.0) : w;
        };
        // this CTA's slice, a contiguous piece of it per warp
        const int slice = (a.V + kDrawCtas - 1) / kDrawCtas, piece = (slice + kDrawWarps - 1) / kDrawWarps;
        const int s_lo = min(a.V, rank * slice), s_hi = min(a.V, s_lo + slice);
        const int w_lo = min(s_hi, s_lo + warp * piece), w_hi = min(s_hi, w_lo + piece);
        double total;
        int round = 0;
        for (;; ++round) {
            double sum = 0.0;
            for (int j = w_lo + lane; j < w_hi; j += 32) sum += left(j);
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == 0) s_warp[warp] = sum;
            __syncthreads();
            if (tid == 0) {
                double mine = 0.0;
                for (int w = 0; w < kDrawWarps; ++w) mine += s_warp[w];
                s_mine[round] = mine;
            }
            cluster_barrier();
            total = 0.0;
            for (int c = 0; c < kDrawCtas; ++c) total += ld_peer(&s_mine[round], c);
            if (total > 0.0 || !residual) break;             // the same in every thread of the cluster
            residual = false;                                // nothing left of p - q: p itself
        }
        // the first CTA, warp and index whose running sum passes `want`; where rounding lets none of them
        // pass it, the last one that weighs anything
        const double want = a.u[(size_t)b * (a.n + 1) + a.n] * total;
        double run = 0.0, before = 0.0;
        int owner = -1;
        for (int c = 0; c < kDrawCtas; ++c) {
            const double part = ld_peer(&s_mine[round], c), next = run + part;
            if (part > 0.0) {
                owner = c;
                before = run;
                if (next > want) break;
            }
            run = next;
        }
        if (owner == rank) {
            int w_own = -1;
            double base = before;
            run = before;
            for (int w = 0; w < kDrawWarps; ++w) {
                const double next = run + s_warp[w];
                if (s_warp[w] > 0.0) {
                    w_own = w;
                    base = run;
                    if (next > want) break;
                }
                run = next;
            }
            if (warp == w_own) {                             // its piece, 32 indices at a time
                int last = -1;
                for (int j0 = w_lo; j0 < w_hi; j0 += 32) {
                    const int j = j0 + lane;
                    const double mine = j < w_hi ? left(j) : 0.0;
                    double v = mine;
                    for (int o = 1; o < 32; o <<= 1) {
                        const double y = __shfl_up_sync(0xffffffffu, v, o);
                        if (lane >= o) v += y;
                    }
                    const unsigned some = __ballot_sync(0xffffffffu, mine > 0.0);
                    const unsigned over = __ballot_sync(0xffffffffu, mine > 0.0 && base + v > want);
                    if (over) {
                        last = j0 + __ffs(over) - 1;
                        break;
                    }
                    if (some) last = j0 + 31 - __clz(some);
                    base += __shfl_sync(0xffffffffu, v, 31);
                }
                if (lane == 0) s_pick = last;
            }
            __syncthreads();
            pick = s_pick;
            write = true;
        }
        cluster_barrier();                                   // the peers have read s_mine
    }
    // write: rank 0 the accepted tokens and the tail, the CTA that found it the drawn one
    int *out = a.out_tokens + (size_t)b * (a.n + 1);
    if (rank == 0) {
        for (int i = tid; i <= a.n; i += kDrawThreads)
            if (i != acc) out[i] = i < acc ? a.tokens[(size_t)b * a.n + i] : -1;
        if (tid == 0) a.accepted[b] = acc;
    }
    if (write && tid == 0) out[acc] = pick;
}

template <typename T>
cudaError_t chains_typed(const ChainArgs &a, cudaStream_t s) {
    ChainStat *st = static_cast<ChainStat *>(a.ws);
    k_chain_stats<T><<<(unsigned)(a.B * chain_rows(a) * chain_chunks(a.V)), kStatThreads, 0, s>>>(a, st);
    k_chain_draw<T><<<a.B * kDrawCtas, kDrawThreads, 0, s>>>(a, st);
    return cudaGetLastError();
}

}  // namespace

size_t chains_workspace(int B, int n, int V) { return (size_t)B * (2 * n + 1) * chain_chunks(V) * sizeof(ChainStat); }

cudaError_t launch_accept_chains(const ChainArgs &a, cudaStream_t s) {
    if (a.type == VT_F32) return chains_typed<float>(a, s);
    return a.type == VT_F16 ? chains_typed<__half>(a, s) : chains_typed<__nv_bfloat16>(a, s);
}

}  // namespace sp
