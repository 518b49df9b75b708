// K / V in pages that requests share: the append of a pass's new keys and values with the position
// rotation on the way, and attention of a ragged batch over a shared prefix and each request's own
// pages (sp_pages_append, sp_pages_attention).
#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>

#include <cuda_bf16.h>

#include "pages.cuh"

namespace sp {

namespace {

// ---- append ----------------------------------------------------------------------------------
// x = qkv + bias; pair (a, b) of a q or k head's first rot dims with (c, s) = table[pos][j]:
// (a c - b s, b c + a s) in fp32, then one rounding to the output's type. Bound by HBM (every byte is
// read and written once) for many tokens, by latency for a decode step. A warp takes one token's
// heads (or, when tokens are few, a slice of them): lane = 16 dims of a head, the two 8-dim halves
// that rotate into each other, so all loads and stores are 16 bytes and the lane's 8 (c, s) pairs
// stay in registers from head to head (32 lanes = 32 / (hd / 16) heads at once, the same dims in
// every round). The token's request is found by a 32-way search of q_start.
// 64 tokens of 28 / 4 heads of 128, fp32: 3.2 us (0.35 at the rate of a copy: one chain of dependent loads). 7,660
// tokens in bf16: 28.8 us, 5.0 TB/s (21.9 at a copy's 6.5). Two rounds of heads under way at once took 96 registers and
// 35.7 us, registers cut to 48 for more warps 31.5, two to nine slices a token 29 to 33.
constexpr int kAppendWarps = 4;

template <typename T>
SP_DEVINL void load8(float (&v)[8], const T *p) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 a = __ldg(reinterpret_cast<const uint4 *>(p));
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) unpack2<T>(w[i], v[2 * i], v[2 * i + 1]);
    }
}
template <typename T>
SP_DEVINL void store8(T *p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint4 a;
        a.x = pack2<T>(v[0], v[1]);
        a.y = pack2<T>(v[2], v[3]);
        a.z = pack2<T>(v[4], v[5]);
        a.w = pack2<T>(v[6], v[7]);
        *reinterpret_cast<uint4 *>(p) = a;
    }
}

// A token's request, own key, position and cache row; false: no such token. A page or length that is
// wrong leaves row < 0 (nothing is written) and the status word set; a position outside the table
// is clamped to it, with the status word set.
SP_DEVINL bool append_place(const PagesAppend &p, int t, int lane, long long &row, int &pos) {
    const PageBatchView &ba = p.ba;
    const int total = ba.q_start ? min(ba.T, ba.q_start[ba.B]) : min((long long)ba.T, (long long)ba.B * ba.max_q);
    if (t >= total) return false;
    const int b = find_request(ba, t, lane);
    const int q0 = request_start(ba, b), qn = request_start(ba, b + 1) - q0;
    const int key = ba.lens[b] - qn + (t - q0);
    row = -1;
    bool bad = key < 0 || key >= (long long)ba.table_width * p.pg.page_size;
    if (!bad) {
        const int pi = key / p.pg.page_size, page = ba.tables[(long long)b * ba.table_stride + pi];
        if ((unsigned)page < (unsigned)p.pg.n_pages)
            row = (long long)page * p.pg.page_stride + (long long)(key - pi * p.pg.page_size) * p.pg.slot_stride;
        else
            bad = true;
    }
    pos = p.pos ? p.pos[t] : ba.prefix_len + key;
    if (pos < 0 || pos >= p.rope_positions) {
        pos = min(max(pos, 0), p.rope_positions - 1);
        bad = true;
    }
    if (bad && lane == 0) set_status(p.pg.status);
    return true;
}

template <typename T, typename TC, int HD>
__global__ void __launch_bounds__(32 * kAppendWarps) k_pages_append(PagesAppend p, int slices) {
    constexpr int UNITS = HD / 16, HEADS = 32 / UNITS;       // lanes per head, heads at once
    const int lane = threadIdx.x & 31;
    const int task = blockIdx.x * kAppendWarps + (threadIdx.x >> 5);
    const int t = task / slices, slice = task - t * slices;
    if (t >= p.ba.T) return;
    long long row;
    int pos;
    if (!append_place(p, t, lane, row, pos)) return;
    const int u = lane % UNITS, nheads = p.nh + 2 * p.pg.nkv;
    // this lane's dims [da, da + 8) and [db, db + 8), and whether they rotate
    const bool turn = p.interleaved ? 16 * u < p.rot : u < p.rot / 16;
    const int r16 = p.rot / 16;
    const int da = p.interleaved || u >= r16 ? 16 * u : 8 * u;
    const int db = p.interleaved || u >= r16 ? 16 * u + 8 : p.rot / 2 + 8 * u;
    float c[8], s[8];
    if (turn) {
        float cs[16];
        const float *tab = p.rope + ((size_t)pos * (p.rot / 2) + 8 * u) * 2;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 f = __ldg(reinterpret_cast<const float4 *>(tab) + i);
            cs[4 * i] = f.x; cs[4 * i + 1] = f.y; cs[4 * i + 2] = f.z; cs[4 * i + 3] = f.w;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) { c[i] = cs[2 * i]; s[i] = cs[2 * i + 1]; }
    }
    const T *x = reinterpret_cast<const T *>(p.x) + (long long)t * p.x_stride;
    T *q = reinterpret_cast<T *>(p.q) + (long long)t * p.q_stride;
    TC *kc = reinterpret_cast<TC *>(p.pg.k), *vc = reinterpret_cast<TC *>(p.pg.v);
    for (int h = slice * HEADS + lane / UNITS; h < nheads; h += slices * HEADS) {
        float a[8], b[8];
        if (p.paired) {                                      // dims d, d + hd / 2 side by side (rot = hd)
            float m0[8], m1[8];
            load8(m0, x + h * HD + 16 * u);
            load8(m1, x + h * HD + 16 * u + 8);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = m0[2 * i]; b[i] = m0[2 * i + 1];
                a[4 + i] = m1[2 * i]; b[4 + i] = m1[2 * i + 1];
            }
        } else {
            load8(a, x + h * HD + da);
            load8(b, x + h * HD + db);
        }
        if (p.bias) {
            float e[8];
            load8(e, p.bias + h * HD + da);
#pragma unroll
            for (int i = 0; i < 8; ++i) a[i] += e[i];
            load8(e, p.bias + h * HD + db);
#pragma unroll
            for (int i = 0; i < 8; ++i) b[i] += e[i];
        }
        if (turn && h < p.nh + p.pg.nkv) {
            if (p.interleaved) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float a0 = a[2 * i], a1 = a[2 * i + 1], b0 = b[2 * i], b1 = b[2 * i + 1];
                    a[2 * i] = a0 * c[i] - a1 * s[i];
                    a[2 * i + 1] = a1 * c[i] + a0 * s[i];
                    b[2 * i] = b0 * c[4 + i] - b1 * s[4 + i];
                    b[2 * i + 1] = b1 * c[4 + i] + b0 * s[4 + i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float a0 = a[i], b0 = b[i];
                    a[i] = a0 * c[i] - b0 * s[i];
                    b[i] = b0 * c[i] + a0 * s[i];
                }
            }
        }
        if (h < p.nh) {
            store8(q + h * HD + da, a);
            store8(q + h * HD + db, b);
        } else if (row >= 0) {
            const int g = h - p.nh;
            TC *dst = g < p.pg.nkv ? kc + row + g * p.pg.head_stride : vc + row + (g - p.pg.nkv) * p.pg.head_stride;
            store8(dst + da, a);
            store8(dst + db, b);
        }
    }
}

// Any rot_dim, stride and alignment: lane = one pair of elements at a time.
template <typename T, typename TC>
__global__ void __launch_bounds__(32 * kAppendWarps) k_pages_append_any(PagesAppend p, int slices) {
    const int lane = threadIdx.x & 31;
    const int task = blockIdx.x * kAppendWarps + (threadIdx.x >> 5);
    const int t = task / slices, slice = task - t * slices;
    if (t >= p.ba.T) return;
    long long row;
    int pos;
    if (!append_place(p, t, lane, row, pos)) return;
    const int hd = p.pg.hd, half = hd / 2, nheads = p.nh + 2 * p.pg.nkv;
    const T *x = reinterpret_cast<const T *>(p.x) + (long long)t * p.x_stride;
    for (int i = slice * 32 + lane; i < nheads * half; i += slices * 32) {
        const int h = i / half, j = i - h * half;
        const bool turn = j < p.rot / 2;
        const int tail = p.rot + 2 * (j - p.rot / 2);        // dims behind the rotated ones, two a lane
        const int da = !turn ? tail : p.interleaved ? 2 * j : j;
        const int db = !turn ? tail + 1 : p.interleaved ? 2 * j + 1 : j + p.rot / 2;
        float a = to_float(x[h * hd + (p.paired ? 2 * j : da)]), b = to_float(x[h * hd + (p.paired ? 2 * j + 1 : db)]);
        if (p.bias) {
            a += p.bias[h * hd + da];
            b += p.bias[h * hd + db];
        }
        if (turn && h < p.nh + p.pg.nkv) {
            const float *cs = p.rope + ((size_t)pos * (p.rot / 2) + j) * 2;
            const float a0 = a, b0 = b;
            a = a0 * cs[0] - b0 * cs[1];
            b = b0 * cs[0] + a0 * cs[1];
        }
        if (h < p.nh) {
            T *q = reinterpret_cast<T *>(p.q) + (long long)t * p.q_stride + h * hd;
            q[da] = from_float<T>(a);
            q[db] = from_float<T>(b);
        } else if (row >= 0) {
            const int g = h - p.nh;
            TC *dst = reinterpret_cast<TC *>(g < p.pg.nkv ? p.pg.k : p.pg.v) + row +
                      (long long)(g < p.pg.nkv ? g : g - p.pg.nkv) * p.pg.head_stride;
            dst[da] = from_float<TC>(a);
            dst[db] = from_float<TC>(b);
        }
    }
}

template <typename T, typename TC>
cudaError_t append_typed(const PagesAppend &p, cudaStream_t s) {
    const auto aligned = [](const void *ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; };
    const long long xs = p.x_stride * (long long)sizeof(T), qs = p.q_stride * (long long)sizeof(T);
    const bool wide = p.rot % 16 == 0 && aligned(p.x) && aligned(p.q) && aligned(p.rope) && (!p.bias || aligned(p.bias)) &&
                      xs % 16 == 0 && qs % 16 == 0;
    const int nheads = p.nh + 2 * p.pg.nkv, hd = p.pg.hd;
    // rounds of 32 lanes a token needs; few tokens: one round a warp, so a decode step's loads are all
    // in flight at once; many: a warp per token, the (c, s) pairs and the search once a token
    const int rounds = wide ? (nheads * (hd / 16) + 31) / 32 : (nheads * (hd / 2) + 31) / 32;
    const int slices = std::max(1, std::min(rounds, (148 * 16 + p.ba.T - 1) / p.ba.T));
    const long long ctas = ((long long)p.ba.T * slices + kAppendWarps - 1) / kAppendWarps;
    if (!wide)
        k_pages_append_any<T, TC><<<(unsigned)ctas, 32 * kAppendWarps, 0, s>>>(p, slices);
    else if (hd == 128)
        k_pages_append<T, TC, 128><<<(unsigned)ctas, 32 * kAppendWarps, 0, s>>>(p, slices);
    else
        k_pages_append<T, TC, 64><<<(unsigned)ctas, 32 * kAppendWarps, 0, s>>>(p, slices);
    return cudaGetLastError();
}

// ---- attention: few rows a kv head ------------------------------------------------------------
// One pass of a key range for at most 16 (query, head) rows of one kv head's group: scores
// S = Q K^T and values O += P V on mma.sync m16n8k16 with fp32 accumulators, online softmax in fp32
// (running maximum and sum per row, exponentials in base 2). Rows are (token, head) pairs of the
// group, row r = token r / G, head r % G: of all requests' tokens for the prefix, so its K and V are
// read once for 16 rows of the batch; of one request's for its own keys. fp32 queries: 8 rows, tile
// row i = fp16 hi of row i's q, 8 + i its fp16 lo, and the probabilities likewise.
// Bound by the K / V stream. Each of the 4 warps walks every fourth tile of 2,048 / HD keys through a
// private ring of shared memory (cp.async, two tiles deep: three CTAs a SM; no block barrier in the loop) and
// keeps its own (m, l, O); the warps' results are joined at the end, the key ranges' by
// k_pages_merge. 64 requests' own keys (35,484 x 4 heads of 128, 73 MB) alone and cold: 24 us (3.0
// TB/s: 257 x 4 CTAs of unequal lengths), with the prefix beside it and the join 37.5; two tiles deep at three CTAs a SM
// beat three tiles at two (by 2 us).
constexpr int kRowsWarps = 4, kRowsStages = 2;
constexpr int kRowsTileBytes = 4096;                         // K (or V) rows of one warp's tile
// Probabilities are held times 2^kRowsBias: at most 2^14, and what fp16's subnormals round off is 2^-39 of the maximum's
// and not 2^-25 (bf16 has fp32's range)
template <typename TC>
constexpr float kRowsBias = std::is_same<TC, __half>::value ? 14.0f : 0.0f;
constexpr int kRowsSmem = kRowsWarps * kRowsStages * 2 * kRowsTileBytes;

template <int HD>
SP_DEVINL uint32_t rows_off(int r, int c) {                  // 16-byte piece c of row r, swizzled
    return (uint32_t)(r * HD * 2 + (((c & ~7) | ((c & 7) ^ (r & 7))) << 4));
}
SP_DEVINL void cp16_zfill(uint32_t dst, const void *src, bool on) {
    const int n = on ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
template <typename TC>
SP_DEVINL void mma16816_t(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<TC, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
SP_DEVINL void ldsm4(uint32_t addr, uint32_t &r0, uint32_t &r1, uint32_t &r2, uint32_t &r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr) : "memory");
}
SP_DEVINL void ldsm4t(uint32_t addr, uint32_t &r0, uint32_t &r1, uint32_t &r2, uint32_t &r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr) : "memory");
}

template <int HD, typename TQ, typename TC>
__global__ void __launch_bounds__(32 * kRowsWarps, 3) k_pages_rows(PagesAttention p, PagesPlan pl) {
    constexpr bool kSplit = sizeof(TQ) == 4;                 // fp32 queries: hi / lo halves
    constexpr int RT = kSplit ? 8 : 16;                      // rows per CTA
    constexpr int KT = kRowsTileBytes / (HD * 2);            // keys per warp tile: 16 or 32
    constexpr int CH = HD / 8, KS = HD / 16, NT = HD / 8, ST = KT / 8;
    extern __shared__ __align__(128) uint8_t smem[];
    const PageBatchView &ba = p.ba;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, tq = lane & 3;
    const int g = blockIdx.y, G = p.nh / p.pg.nkv;
    griddep_launch_dependents();
    if (pl.prefix_tc || pl.own_tc) {
        // beside k_pages_tc: the last CTA ends after that grid, so that the join, which waits for this one, waits
        // for both
        if (blockIdx.x == gridDim.x - 1) {
            if (blockIdx.y == 0) griddep_wait();
            return;
        }
    }
    // the item: its rows, its key range and its pages
    const int n_prefix = pl.prefix_tc ? 0 : pl.prefix_tiles * pl.prefix_splits;
    const int total = total_rows(ba);
    int item = blockIdx.x, row0, nrows, q0 = 0, own0 = INT_MAX / 2, slot, k_lo, k_hi, k_own = 0;
    const int *table, *table_own = nullptr;                  // keys [k_lo, k_hi) of table, then [0, k_own) of table_own
    if (item < n_prefix) {
        slot = item / pl.prefix_tiles;
        row0 = (item - slot * pl.prefix_tiles) * RT;
        nrows = min(RT, total * G - row0);
        k_lo = slot * pl.prefix_chunk;
        k_hi = min(ba.prefix_len, k_lo + pl.prefix_chunk);
        table = ba.prefix;
        if (nrows <= 0) return;
    } else {
        item -= n_prefix;
        const int per = pl.own_tiles * (pl.whole ? 1 : pl.own_splits), b = item / per;
        item -= b * per;
        const int z = item / pl.own_tiles;
        slot = pl.prefix_slots + z;
        q0 = request_start(ba, b);
        const int qn = min(request_start(ba, b + 1), total) - q0, len = own_len(p, b, lane);
        row0 = (item - z * pl.own_tiles) * RT;
        nrows = min(RT, qn * G - row0);
        own0 = len - qn;                                     // token 0's own key
        if (qn > ba.max_q && threadIdx.x == 0) set_status(p.pg.status);
        int chunk = 0, n = 1;
        if (!pl.whole) own_chunks(len, pl.own_splits, chunk, n);
        if (nrows <= 0) return;
        if (z >= n) {                                        // no such range: nothing to join
            if (threadIdx.x < nrows) {
                const int row = row0 + threadIdx.x;
                const long long at = ((long long)slot * ba.T + q0 + row / G) * p.nh + g * G + row % G;
                *reinterpret_cast<float2 *>(pl.ml + at * 2) = make_float2(-INFINITY, 0.f);
            }
            return;
        }
        const int last = min(len, own0 + (row0 + nrows - 1) / G + 1);
        table_own = ba.tables + (long long)b * ba.table_stride;
        if (pl.whole) {
            table = ba.prefix;
            k_lo = 0;
            k_hi = ba.prefix_len;
            k_own = max(0, last);
        } else {
            table = table_own;
            k_lo = z * chunk;
            k_hi = min(k_lo + chunk, last);
        }
    }
    const int ntiles0 = k_hi > k_lo ? (k_hi - k_lo + KT - 1) / KT : 0, ntiles = ntiles0 + (k_own + KT - 1) / KT;
    const bool own = table == table_own;                     // the first keys are the request's own
    const TC *kb = reinterpret_cast<const TC *>(p.pg.k) + g * p.pg.head_stride;
    const TC *vbase = reinterpret_cast<const TC *>(p.pg.v) + g * p.pg.head_stride;
    const uint32_t ring = smem_u32(smem) + warp * (kRowsStages * 2 * kRowsTileBytes);
    // The page numbers of 32 pages of the walk, a lane each, so that no tile waits for its own. Pages of whole
    // tiles (the usual case): a tile's rows are slot_stride apart; else every row looks its page up.
    const int ps = p.pg.page_size;
    const bool whole_tiles = ps % KT == 0;
    int win_first = 0, win_end = 0, win = 0;                 // pages [win_first, win_first + 32) of the keys below win_end
    const auto fill_window = [&](const int *tab, int first, int hi) {
        win_first = first;
        win_end = hi;
        const long long key0 = (long long)(first + lane) * ps;
        win = key0 < hi ? __ldg(tab + first + lane) : 0;
    };
    bool win_own = false;
    // a key's row in its page, -1 on a bad page number (uniform arguments: the window may move)
    const auto row_at = [&](int key, int page) -> long long {
        if ((unsigned)page >= (unsigned)p.pg.n_pages) {
            set_status(p.pg.status);
            return -1;
        }
        return (long long)page * p.pg.page_stride + (long long)(key % ps) * p.pg.slot_stride;
    };
    const long long lane_off = (long long)(lane / CH) * p.pg.slot_stride + (lane % CH) * 8;
    const auto stage = [&](int tile) {
        const uint32_t ks = ring + (uint32_t)((tile / kRowsWarps) % kRowsStages) * 2 * kRowsTileBytes;
        const uint32_t vs = ks + kRowsTileBytes;
        const bool second = tile >= ntiles0;
        const int key0 = second ? (tile - ntiles0) * KT : k_lo + tile * KT, hi = second ? k_own : k_hi;
        const int *tab = second ? table_own : table;
        if (tile < ntiles && whole_tiles) {
            const int pi = key0 / ps;
            if (second != win_own || win_end == 0 || pi > win_first + 31) {
                win_own = second;
                fill_window(tab, pi, hi);
            }
            const long long row = row_at(key0, __shfl_sync(0xffffffffu, win, pi - win_first));
            const TC *kp = kb + (row < 0 ? 0 : row + lane_off), *vp = vbase + (row < 0 ? 0 : row + lane_off);
            const long long step = row < 0 ? 0 : 32 / CH * p.pg.slot_stride;
            const int left = row < 0 ? 0 : hi - key0 - lane / CH;    // of the lane's rows, every 32 / CH-th
#pragma unroll
            for (int i = 0; i < KT * CH / 32; ++i) {
                const uint32_t at = rows_off<HD>(i * (32 / CH) + lane / CH, lane % CH);
                const bool on = i * (32 / CH) < left;
                cp16_zfill(ks + at, on ? kp + i * step : kb, on);
                cp16_zfill(vs + at, on ? vp + i * step : vbase, on);
            }
        } else if (tile < ntiles) {
            const int key = min(key0 + min(lane, KT - 1), hi - 1), pi = key / ps, last = min(key0 + KT, hi) - 1;
            if (second != win_own || win_end == 0 || last / ps > win_first + 31) {
                win_own = second;
                fill_window(tab, key0 / ps, hi);
            }
            const long long row = row_at(key, __shfl_sync(0xffffffffu, win, pi - win_first));
#pragma unroll
            for (int i = 0; i < KT * CH / 32; ++i) {
                const int r = i * (32 / CH) + lane / CH;
                const long long o = __shfl_sync(0xffffffffu, row, r);
                const uint32_t at = rows_off<HD>(r, lane % CH);
                const bool on = o >= 0 && key0 + r < hi;
                cp16_zfill(ks + at, on ? kb + o + lane % CH * 8 : kb, on);
                cp16_zfill(vs + at, on ? vbase + o + lane % CH * 8 : vbase, on);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kRowsStages - 1; ++i) stage(warp + i * kRowsWarps);
    // q fragments: tile rows gq and gq + 8 at dims 16 kk + 2 tq + {0, 1} and + 8
    uint32_t qa[KS][4];
    const int ra = row0 + gq, rb = kSplit ? ra : row0 + gq + 8;
    const bool la = gq < nrows, lb = kSplit ? la : gq + 8 < nrows;
    const TQ *qbase = reinterpret_cast<const TQ *>(p.q);
    const auto q_row = [&](int r) { return qbase + (long long)(q0 + r / G) * p.q_stride + (g * G + r % G) * HD; };
    float up = 1.f;                                          // fp32 queries: what the row's were divided by
    {
        const TQ *pa = q_row(la ? ra : row0), *pb = q_row(lb ? rb : row0);
        float down = 1.f;
        float2 xs[kSplit ? 2 * KS : 1];                      // at dims 8 i + 2 tq
        if constexpr (kSplit) {
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < 2 * KS; ++i) {
                xs[i] = la ? *reinterpret_cast<const float2 *>(pa + 8 * i + 2 * tq) : make_float2(0.f, 0.f);
                top = fmaxf(top, fmaxf(fabsf(xs[i].x), fabsf(xs[i].y)));
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            row_power(top, down, up);
        }
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const int d = 16 * kk + 8 * hf + 2 * tq;
                if constexpr (kSplit) {
                    const float2 x = make_float2(xs[2 * kk + hf].x * down, xs[2 * kk + hf].y * down);
                    const __half ha = __float2half_rn(x.x), hb = __float2half_rn(x.y);
                    qa[kk][2 * hf] = pack2<__half>(x.x, x.y);
                    qa[kk][2 * hf + 1] = pack2<__half>(x.x - __half2float(ha), x.y - __half2float(hb));
                } else {
                    qa[kk][2 * hf] = la ? *reinterpret_cast<const uint32_t *>(pa + d) : 0u;
                    qa[kk][2 * hf + 1] = lb ? *reinterpret_cast<const uint32_t *>(pb + d) : 0u;
                }
            }
        }
    }
    // own keys each row sees: below this
    const int sa = own0 + ra / G + 1, sb = own0 + rb / G + 1;
    const float sc = kSplit ? row_scale(p, up) : row_scale(p);
    float o[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    for (int tile = warp; tile < ntiles; tile += kRowsWarps) {
        stage(tile + (kRowsStages - 1) * kRowsWarps);
        asm volatile("cp.async.wait_group %0;" ::"n"(kRowsStages - 1) : "memory");
        __syncwarp();
        const uint32_t ks = ring + (uint32_t)((tile / kRowsWarps) % kRowsStages) * 2 * kRowsTileBytes;
        const uint32_t vs = ks + kRowsTileBytes;
        // the tile's keys that each row sees: below va, vb
        const bool second = tile >= ntiles0;
        const int j0 = second ? (tile - ntiles0) * KT : k_lo + tile * KT, hi = second ? k_own : k_hi;
        const int va = own || second ? min(hi, sa) : hi, vb = own || second ? min(hi, sb) : hi;
        float s[ST][4];
#pragma unroll
        for (int nt = 0; nt < ST; ++nt) {
            s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
            for (int kk = 0; kk < KS; kk += 2) {
                uint32_t b0, b1, b2, b3;
                ldsm4(ks + rows_off<HD>(8 * nt + (lane & 7), 2 * kk + (lane >> 3)), b0, b1, b2, b3);
                mma16816_t<TC>(s[nt], qa[kk], b0, b1);
                mma16816_t<TC>(s[nt], qa[kk + 1], b2, b3);
            }
        }
        // mask, running maximum (kSplit: both tile rows are one row)
        float mt[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int nt = 0; nt < ST; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int key = j0 + 8 * nt + 2 * tq + e;
                if constexpr (kSplit) s[nt][e] += s[nt][2 + e];
                s[nt][e] = key < va ? s[nt][e] : -INFINITY;
                mt[0] = fmaxf(mt[0], s[nt][e]);
                if constexpr (!kSplit) {
                    s[nt][2 + e] = key < vb ? s[nt][2 + e] : -INFINITY;
                    mt[1] = fmaxf(mt[1], s[nt][2 + e]);
                }
            }
        }
        float corr[2] = {1.f, 1.f}, ms[2];
        constexpr int NR = kSplit ? 1 : 2;
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            mt[i] = fmaxf(mt[i], __shfl_xor_sync(0xffffffffu, mt[i], 1));
            mt[i] = fmaxf(mt[i], __shfl_xor_sync(0xffffffffu, mt[i], 2));
            const float mn = fmaxf(m[i], mt[i]);
            ms[i] = mn == -INFINITY ? 0.f : mn;              // a row that has seen no key yet
            corr[i] = exp2_approx((m[i] - ms[i]) * sc);
            m[i] = mn;
            l[i] *= corr[i];
        }
        if constexpr (kSplit) corr[1] = corr[0];
        if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                o[n][0] *= corr[0];
                o[n][1] *= corr[0];
                o[n][2] *= corr[1];
                o[n][3] *= corr[1];
            }
        }
        uint32_t pa[ST / 2][4];
#pragma unroll
        for (int nt = 0; nt < ST; ++nt) {
            float e[4];
#pragma unroll
            for (int i = 0; i < 2 * NR; ++i) e[i] = exp2_approx(fmaf(s[nt][i] - ms[i >> 1], sc, kRowsBias<TC>));
            l[0] += e[0] + e[1];
            uint32_t hi = pack2<TC>(e[0], e[1]), lo;
            if constexpr (kSplit) {
                float h0, h1;
                unpack2<TC>(hi, h0, h1);
                lo = pack2<TC>(e[0] - h0, e[1] - h1);
            } else {
                l[1] += e[2] + e[3];
                lo = pack2<TC>(e[2], e[3]);
            }
            pa[nt >> 1][2 * (nt & 1)] = hi;
            pa[nt >> 1][2 * (nt & 1) + 1] = lo;
        }
#pragma unroll
        for (int kk = 0; kk < ST / 2; ++kk) {
#pragma unroll
            for (int n = 0; n < NT; n += 2) {
                uint32_t b0, b1, b2, b3;
                const int mtx = lane >> 3;
                ldsm4t(vs + rows_off<HD>(16 * kk + 8 * (mtx & 1) + (lane & 7), n + (mtx >> 1)), b0, b1, b2, b3);
                mma16816_t<TC>(o[n], pa[kk], b0, b1);
                mma16816_t<TC>(o[n + 1], pa[kk], b2, b3);
            }
        }
        __syncwarp();                                        // the stage is rewritten by the next round
    }
    // the warps' (m, l, O) through shared memory (the rings are done)
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    __syncthreads();
    constexpr int OS = HD + 4;                               // row stride of the joined O, floats
    float *so = reinterpret_cast<float *>(smem), *sm = so + kRowsWarps * RT * OS;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float *d = so + (warp * RT + gq) * OS + 8 * n + 2 * tq;
        if constexpr (kSplit) {
            *reinterpret_cast<float2 *>(d) = make_float2(o[n][0] + o[n][2], o[n][1] + o[n][3]);
        } else {
            *reinterpret_cast<float2 *>(d) = make_float2(o[n][0], o[n][1]);
            *reinterpret_cast<float2 *>(d + 8 * OS) = make_float2(o[n][2], o[n][3]);
        }
    }
    if (tq == 0) {
        sm[(warp * RT + gq) * 2] = m[0] * up;
        sm[(warp * RT + gq) * 2 + 1] = l[0];
        if constexpr (!kSplit) {
            sm[(warp * RT + gq + 8) * 2] = m[1];
            sm[(warp * RT + gq + 8) * 2 + 1] = l[1];
        }
    }
    __syncthreads();
    constexpr int TPR = 32 * kRowsWarps / RT, DPT = HD / TPR;  // threads per row, dims per thread
    const int r = threadIdx.x / TPR, d0 = (threadIdx.x % TPR) * DPT;
    if (r >= nrows) return;
    float M = -INFINITY, L = 0.f, acc[DPT];
#pragma unroll
    for (int w = 0; w < kRowsWarps; ++w) M = fmaxf(M, sm[(w * RT + r) * 2]);
    const float Ms = M == -INFINITY ? 0.f : M, c = kSplit ? row_scale(p) : sc;    // this row's own
#pragma unroll
    for (int d = 0; d < DPT; ++d) acc[d] = 0.f;
#pragma unroll
    for (int w = 0; w < kRowsWarps; ++w) {
        const float f = exp2_approx(fmaf(sm[(w * RT + r) * 2] - Ms, c, -kRowsBias<TC>));
        L = fmaf(sm[(w * RT + r) * 2 + 1], f, L);
#pragma unroll
        for (int d = 0; d < DPT; ++d) acc[d] = fmaf(so[(w * RT + r) * OS + d0 + d], f, acc[d]);
    }
    const long long rt = q0 + (row0 + r) / G, hh = g * G + (row0 + r) % G;
    if (pl.slots == 1) {
        const float inv = L > 0.f ? 1.f / L : 0.f;
        TQ *dst = reinterpret_cast<TQ *>(p.out) + rt * p.out_stride + hh * HD + d0;
#pragma unroll
        for (int d = 0; d < DPT; ++d) dst[d] = from_float<TQ>(L == L ? acc[d] * inv : L);
        if (p.lse && d0 == 0) p.lse[rt * p.nh + hh] = row_lse(M, L, c);
    } else {
        const long long at = ((long long)slot * ba.T + rt) * p.nh + hh;
        float *dst = pl.acc + at * HD + d0;
#pragma unroll
        for (int d = 0; d < DPT; d += 4) *reinterpret_cast<float4 *>(dst + d) = make_float4(acc[d], acc[d + 1], acc[d + 2], acc[d + 3]);
        if (d0 == 0) *reinterpret_cast<float2 *>(pl.ml + at * 2) = make_float2(M, L);
    }
}

// The key ranges' partials of a (token, head): a CTA, warp w the slots w, w + 4, .., lane = HD / 32 dims. Every
// slot's (m, l) is read at once, so that the partials' loads depend on nothing else and 8 a lane are on their
// way; a slot without weight (a range that does not exist) is passed over. The warps' sums are added in order. Bound
// by latency: 1,792 (token, heads) of up to 20 slots alone and cold 9.7 us, 18 MB.
constexpr int kMergeWarps = 4;
constexpr int kMergeSlots = 4 * kPagesMaxSplits;
constexpr int kMergeFew = 32, kMergeFewCtas = 148 * 16;
template <int HD, typename TQ>
__global__ void __launch_bounds__(32 * kMergeWarps) k_pages_merge(PagesAttention p, PagesPlan pl) {
    constexpr int DL = HD / 32, NS = kMergeSlots / 32, BATCH = 8;
    __shared__ float s_w[kMergeSlots];
    __shared__ float s_acc[kMergeWarps][HD];
    const PageBatchView &ba = p.ba;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int t = blockIdx.x / p.nh, h = blockIdx.x - t * p.nh;
    const bool none = t >= total_rows(ba);
    griddep_wait();                                          // every CTA: the next grid in the stream starts after all of them
    if (none) return;
    const long long step = (long long)ba.T * p.nh, at = blockIdx.x;
    float2 ml[NS];
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int s = 32 * i + lane;
        ml[i] = make_float2(-INFINITY, 0.f);
        if (s < pl.slots) ml[i] = *reinterpret_cast<const float2 *>(pl.ml + (s * step + at) * 2);
        M = fmaxf(M, ml[i].x);
    }
    M = warp_max(M);
    const float Ms = M == -INFINITY ? 0.f : M, sc = row_scale(p);
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const float f = exp2_approx((ml[i].x - Ms) * sc);
        L = fmaf(ml[i].y, f, L);
        if (warp == 0) s_w[32 * i + lane] = f;
    }
    L = warp_sum(L);                                         // the same bits in every warp
    __syncthreads();
    float acc[DL];
#pragma unroll
    for (int d = 0; d < DL; ++d) acc[d] = 0.f;
    for (int s0 = warp; s0 < pl.slots; s0 += kMergeWarps * BATCH) {
        float f[BATCH], v[BATCH][DL];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int s = s0 + kMergeWarps * i;
            f[i] = s < pl.slots ? s_w[s] : 0.f;
#pragma unroll
            for (int d = 0; d < DL; ++d) v[i][d] = 0.f;
            if (!(f[i] == 0.f)) {
                const float *src = pl.acc + (s * step + at) * HD + lane * DL;
                if constexpr (DL == 4) {
                    const float4 x = *reinterpret_cast<const float4 *>(src);
                    v[i][0] = x.x;
                    v[i][1] = x.y;
                    v[i][2] = x.z;
                    v[i][3] = x.w;
                } else {
                    const float2 x = *reinterpret_cast<const float2 *>(src);
                    v[i][0] = x.x;
                    v[i][1] = x.y;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
#pragma unroll
            for (int d = 0; d < DL; ++d) acc[d] = fmaf(v[i][d], f[i], acc[d]);
    }
#pragma unroll
    for (int d = 0; d < DL; ++d) s_acc[warp][lane * DL + d] = acc[d];
    __syncthreads();
    const float inv = L > 0.f ? 1.f / L : 0.f;
    for (int d = threadIdx.x; d < HD; d += 32 * kMergeWarps) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kMergeWarps; ++w) v += s_acc[w][d];
        reinterpret_cast<TQ *>(p.out)[(long long)t * p.out_stride + h * HD + d] = from_float<TQ>(L == L ? v * inv : L);
    }
    if (p.lse && threadIdx.x == 0) p.lse[at] = row_lse(M, L, sc);
}

// The same with a warp per (token, head), for at most 32 ranges: no shared memory, no barrier. Where a CTA per (token,
// head) no longer has them all on the GPU at once: with their attention, 3,976 (token, heads)
// of 11 ranges 50.2 -> 46.1 us, 22,400 of 2 118 -> 96; but 1,792 of 20 39.1 -> 39.9.
template <int HD, typename TQ>
__global__ void __launch_bounds__(32 * kMergeWarps) k_pages_merge_few(PagesAttention p, PagesPlan pl) {
    constexpr int DL = HD / 32, BATCH = 8;
    const PageBatchView &ba = p.ba;
    const int lane = threadIdx.x & 31;
    const long long step = (long long)ba.T * p.nh, at = (long long)blockIdx.x * kMergeWarps + (threadIdx.x >> 5);
    const int t = (int)(at / p.nh), h = (int)(at - (long long)t * p.nh);
    const bool none = t >= total_rows(ba);
    griddep_wait();
    if (none) return;
    const float2 ml = lane < pl.slots ? *reinterpret_cast<const float2 *>(pl.ml + (lane * step + at) * 2) : make_float2(-INFINITY, 0.f);
    const float M = warp_max(ml.x), sc = row_scale(p), w = exp2_approx((ml.x - (M == -INFINITY ? 0.f : M)) * sc);
    const float L = warp_sum(ml.y * w);
    float acc[DL];
#pragma unroll
    for (int d = 0; d < DL; ++d) acc[d] = 0.f;
    for (int s0 = 0; s0 < pl.slots; s0 += BATCH) {
        float f[BATCH], v[BATCH][DL];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            f[i] = __shfl_sync(0xffffffffu, w, s0 + i);          // 0 behind the last
#pragma unroll
            for (int d = 0; d < DL; ++d) v[i][d] = 0.f;
            if (!(f[i] == 0.f)) {
                const float *src = pl.acc + ((s0 + i) * step + at) * HD + lane * DL;
                if constexpr (DL == 4) {
                    const float4 x = *reinterpret_cast<const float4 *>(src);
                    v[i][0] = x.x;
                    v[i][1] = x.y;
                    v[i][2] = x.z;
                    v[i][3] = x.w;
                } else {
                    const float2 x = *reinterpret_cast<const float2 *>(src);
                    v[i][0] = x.x;
                    v[i][1] = x.y;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
#pragma unroll
            for (int d = 0; d < DL; ++d) acc[d] = fmaf(v[i][d], f[i], acc[d]);
    }
    const float inv = L > 0.f ? 1.f / L : 0.f;
    TQ *dst = reinterpret_cast<TQ *>(p.out) + (long long)t * p.out_stride + h * HD + lane * DL;
#pragma unroll
    for (int d = 0; d < DL; ++d) acc[d] = L == L ? acc[d] * inv : L;
    if constexpr (sizeof(TQ) == 4) {
        if constexpr (DL == 4) *reinterpret_cast<float4 *>(dst) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        else *reinterpret_cast<float2 *>(dst) = make_float2(acc[0], acc[1]);
    } else {
        if constexpr (DL == 4) *reinterpret_cast<uint2 *>(dst) = make_uint2(pack2<TQ>(acc[0], acc[1]), pack2<TQ>(acc[2], acc[3]));
        else *reinterpret_cast<uint32_t *>(dst) = pack2<TQ>(acc[0], acc[1]);
    }
    if (p.lse && lane == 0) p.lse[at] = row_lse(M, L, sc);
}

// Which kernel takes what. k_pages_tc pads a row tile to 128 rows and needs an SM to itself; k_pages_rows reads K and
// V again for every 16 rows (8 with fp32 queries).
constexpr int kSms = 148;
// The prefix: up to 32 rows a kv head by k_pages_rows (28 rows of 4 heads over 4,096 keys 13.0 against 14.6 us, over
// 16,384 20.5 against 21.2), more by k_pages_tc once the reads beyond those of 32 rows pass so many bytes (35 rows over
// 4,096 keys, 8 MB: 13.4 against 14.6; over 16,384, 34 MB: 28.8 against 21.3; fp32, 25 MB: 15.7 against 18.3, 34 MB:
// 33.3 against 29.2).
constexpr int kTcMinRows = 32;
constexpr double kRowsReads = 12e6, kF32RowsReads = 28e6;
// A request's own keys: by k_pages_tc from more rows than this on (8 requests of 84 rows 31.0 against 35.5 us, of 42
// 24.2 against 23.8; fp32, of 126 47.4 against 49.7, of 63 37.2 against 31.4).
constexpr int kTcMinOwnRows = 64;
constexpr int kWholeValues = 40960, kWholeCtas = 2 * kSms;
// measured on k_pages_tc: a CTA's start and end, a key tile of two row tiles, of one (the alternate walk), and
// k_pages_rows' rate over own keys
constexpr double kTcFixedUs = 8.0, kTcTileUs = 1.8, kTcAltTileUs = 1.0, kOwnBytesPerUs = 4.5e6;
// Many rows a request: one walk over the prefix and the own keys, or parts that are joined. Fitted to 49 sizes (rows
// 420 to 11,200, prefixes of 60 to 4,000 keys; the times within 5 and 8 %): a walk's start and end and its key tile,
// as many rounds of them as the SMs need; the parts' start and join, a key tile's share of all SMs, the partials'
// rate. 8 requests of 100 tokens, 4,000 keys: 80 us in one walk, 96 in parts; 4 requests: 79 and 59.
constexpr double kWalkFixedUs = 13.0, kWalkTileUs = 2.0, kF32WalkTileUs = 3.0, kPartsFixedUs = 14.0, kPartsTileUs = 2.8,
                 kJoinBytesPerUs = 3e6;
constexpr int kF32TcKeys = 4096, kF32RowsKeys = 4096;
constexpr int kOwnCtas = 8 * kSms;           // k_pages_rows' CTAs over own keys: requests differ in length
PagesPlan plan_attention(const PagesAttention &p) {
    PagesPlan pl{};
    const PageBatchView &ba = p.ba;
    const auto up = [](long long a, long long b) { return (a + b - 1) / b; };
    const bool f32 = p.q_type == VT_F32, fits = pages_tc_fits(p.pg);
    const int G = p.nh / p.pg.nkv, rt = f32 ? 8 : 16, nkv = p.pg.nkv;
    const long long rows = (long long)ba.T * G, own_rows = (long long)std::min(ba.max_q, ba.T) * G;
    const long long bound = (long long)ba.table_width * p.pg.page_size;
    const int pair = f32 ? 128 : 256;                        // rows of a k_pages_tc CTA that needs no partner
    // few requests and a walk of at most 5 tiles a warp: one launch and no join (4 requests, 602 keys of 64
    // dims: 8.0 us on the GPU against 6.9 in two launches, but 10.2 a call in a loop against 13.0)
    const long long small_tiles = up(own_rows, rt);
    if (ba.prefix_len > 0 && (ba.prefix_len + bound) * p.pg.hd <= kWholeValues && ba.B * small_tiles * nkv <= kWholeCtas) {
        pl.whole = 1;
        pl.own_tiles = (int)small_tiles;
        pl.slots = 1;
        return pl;
    }
    // key ranges that fill the GPU; fp32 queries: no longer than `most` (what the MMAs' accumulators cut off), up to
    // kPagesMaxSplits ranges
    const auto splits = [&](long long ctas, long long want, long long keys, long long most) {
        const long long least = f32 ? up(keys, most) : 1;
        return std::min<long long>({std::max<long long>(least, want / ctas), up(keys, kPagesOwnKeys), kPagesMaxSplits});
    };
    if (bound > 0) {
        pl.own_tc = fits && own_rows > kTcMinOwnRows;
        pl.own_alt = pl.own_tc && (f32 || own_rows <= 128);
        pl.own_tiles = (int)up(own_rows, !pl.own_tc ? rt : pl.own_alt ? 128 : 256);
        pl.own_splits = (int)splits((long long)ba.B * pl.own_tiles * nkv, pl.own_tc ? kSms : kOwnCtas, bound, pl.own_tc ? kF32TcKeys : kF32RowsKeys);
    }
    if (ba.prefix_len > 0) {
        const double read = (double)ba.prefix_len * nkv * p.pg.hd * 4;
        pl.prefix_tc = fits && rows > kTcMinRows && (pl.own_tc || (up(rows, rt) - kTcMinRows / rt) * read > (f32 ? kF32RowsReads : kRowsReads));
        pl.prefix_alt = pl.prefix_tc && (f32 || rows <= 128);
        pl.prefix_tiles = (int)up(rows, !pl.prefix_tc ? rt : pl.prefix_alt ? 128 : 256);
        const long long row_ctas = (long long)pl.prefix_tiles * nkv;
        long long n = splits(row_ctas, pl.prefix_tc ? kSms : 2 * kSms, ba.prefix_len, pl.prefix_tc ? kF32TcKeys : kF32RowsKeys);
        const long long least = f32 ? std::min<long long>(n, up(ba.prefix_len, kF32TcKeys)) : 1;
        if (pl.prefix_tc) {
            // k_pages_tc shares the GPU with the own keys' kernel: the fewest ranges that take no longer than
            // both kernels' work spread over all SMs (in us; own keys: half the tables' capacity)
            const double own_us = pl.own_tc ? 0.0 : 0.5 * (double)(ba.B * bound) * nkv * p.pg.hd * 4 * pl.own_tiles / kOwnBytesPerUs;
            const double tiles = (double)up(ba.prefix_len, 128), tile_us = pl.prefix_alt ? kTcAltTileUs : kTcTileUs;
            double best = 1e30;
            for (long long k = n, most = n; k >= least; --k) {
                const double t = kTcFixedUs + std::ceil(tiles / k) * tile_us;
                const double all = std::max(t, (double)(k * row_ctas) / kSms * t + own_us);
                if (all <= best * (k == most ? 1.0 : 0.999)) {
                    best = all;
                    n = k;
                }
            }
        }
        pl.prefix_chunk = (int)(up(up(ba.prefix_len, n), kPagesGrain) * kPagesGrain);
        pl.prefix_splits = (int)up(ba.prefix_len, pl.prefix_chunk);
        pl.prefix_slots = pl.prefix_splits << pl.prefix_alt;
    }
    pl.slots = pl.prefix_slots + (pl.own_splits << pl.own_alt);
    // many rows a request: the prefix and the own keys in one walk, no partials
    if (fits && bound > 0 && own_rows > 128) {
        const long long tiles = up(own_rows, pair), items = std::min<long long>(ba.B * tiles, up(rows, pair) + ba.B / 2) * nkv;
        const double prefix = (double)up(ba.prefix_len, 128), own = 0.5 * (double)up(bound, 128);
        const double scale = f32 && p.pg.hd == 64 ? 0.7 : 1.0;
        const double one = up(items, kSms) * (kWalkFixedUs + (prefix + own) * (f32 ? kF32WalkTileUs : kWalkTileUs) * scale);
        const double parts = kPartsFixedUs + ((double)(up(rows, pair) * nkv) * prefix + items * own) * kPartsTileUs * scale / kSms +
                             (double)ba.T * p.nh * p.pg.hd * 8 * pl.slots / kJoinBytesPerUs;
        if (one <= parts) {
            pl = PagesPlan{};
            pl.whole = pl.own_tc = 1;
            pl.own_tiles = (int)tiles;
            pl.slots = 1;
        }
    }
    return pl;
}
size_t plan_bytes(const PagesAttention &p, const PagesPlan &pl) {
    return pl.slots <= 1 ? 0 : (size_t)pl.slots * p.ba.T * p.nh * (p.pg.hd + 2) * sizeof(float);
}

template <int HD, typename TQ, typename TC>
cudaError_t attention_typed(const PagesAttention &p, PagesPlan pl, cudaStream_t s) {
    const int nkv = p.pg.nkv;
    pl.acc = static_cast<float *>(p.ws);
    pl.ml = pl.acc + (size_t)pl.slots * p.ba.T * p.nh * HD;
    if (pl.prefix_tc || pl.own_tc) {
        const cudaError_t e = launch_pages_tc(p, pl, s);
        if (e != cudaSuccess || pl.whole) return e;
    }
    const int items = (pl.prefix_tc ? 0 : pl.prefix_tiles * pl.prefix_splits) +
                      (pl.own_tc ? 0 : p.ba.B * pl.own_tiles * (pl.whole ? 1 : pl.own_splits));
    cudaError_t e = raise_smem(k_pages_rows<HD, TQ, TC>, kRowsSmem);
    if (e != cudaSuccess) return e;
    // k_pages_rows does not read what k_pages_tc writes: it starts beside it (and ends after it, which is what
    // the join waits for)
    if (items > 0) {
        if (pl.prefix_tc || pl.own_tc)
            e = launch_dependent(k_pages_rows<HD, TQ, TC>, dim3(items + 1, nkv), 32 * kRowsWarps, kRowsSmem, s, p, pl);
        else
            k_pages_rows<HD, TQ, TC><<<dim3(items, nkv), 32 * kRowsWarps, kRowsSmem, s>>>(p, pl);
    }
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e == cudaSuccess && pl.slots == 0)                   // no keys at all: zeros, and nothing to start beside
        k_pages_merge<HD, TQ><<<(unsigned)(p.ba.T * p.nh), 32 * kMergeWarps, 0, s>>>(p, pl);
    else if (e == cudaSuccess && pl.slots > 1 && pl.slots <= kMergeFew && p.ba.T * p.nh > kMergeFewCtas)
        e = launch_dependent(k_pages_merge_few<HD, TQ>, dim3((unsigned)((p.ba.T * p.nh + kMergeWarps - 1) / kMergeWarps)),
                             32 * kMergeWarps, 0, s, p, pl);
    else if (e == cudaSuccess && pl.slots != 1)
        e = launch_dependent(k_pages_merge<HD, TQ>, dim3((unsigned)(p.ba.T * p.nh)),
                             32 * kMergeWarps, 0, s, p, pl);
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace

cudaError_t launch_pages_append(const PagesAppend &p, cudaStream_t s) {
    if (p.ba.T == 0) return cudaSuccess;
    if (p.in_type == VT_F32)
        return p.cache_type == VT_F16 ? append_typed<float, __half>(p, s) : append_typed<float, __nv_bfloat16>(p, s);
    return p.in_type == VT_F16 ? append_typed<__half, __half>(p, s) : append_typed<__nv_bfloat16, __nv_bfloat16>(p, s);
}

size_t pages_attention_workspace(const PagesAttention &p) { return plan_bytes(p, plan_attention(p)); }

cudaError_t launch_pages_attention(const PagesAttention &p, cudaStream_t s) {
    if (p.ba.T == 0) return cudaSuccess;
    const PagesPlan pl = plan_attention(p);
    const bool wide = p.pg.hd == 128;
    if (p.q_type == VT_F32)
        return wide ? attention_typed<128, float, __half>(p, pl, s) : attention_typed<64, float, __half>(p, pl, s);
    if (p.q_type == VT_F16)
        return wide ? attention_typed<128, __half, __half>(p, pl, s) : attention_typed<64, __half, __half>(p, pl, s);
    return wide ? attention_typed<128, __nv_bfloat16, __nv_bfloat16>(p, pl, s)
                : attention_typed<64, __nv_bfloat16, __nv_bfloat16>(p, pl, s);
}

}  // namespace sp
