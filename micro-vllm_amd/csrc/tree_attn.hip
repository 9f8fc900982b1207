// Attention for trees of drafted tokens over the paged cache: node i of row b (tree_ops.hip) sees the row's ctx cached tokens and
// the nodes whose bits its mask has, o = sum_j softmax_j(q . k_j scale) v_j.  The nodes' own keys and values are in the cache already.
//
// The g query heads that share a key/value head are stacked: stacked row r = node * g + head, so every key read serves n * g rows.
// Workgroup = (row, key/value head, run of stacked rows, split of the keys), one pass over the keys with a softmax state per stacked row.
// Three forms: fp32 and bf16 with few rows, where every wave takes blocks of keys of its own and the states meet in LDS at the end, and bf16 with many
// rows, where the waves share the keys.  The splits' states are added in order by a second launch.
#include "common.h"

#include <type_traits>

namespace mv {

constexpr float kTreeNegBig = -3.4028235e38f;  // a running maximum before any visible key: below any score
// A row's running maximum is raised only when a score outgrows it by this many powers of two: weights are then up to 2^6 instead of up to
// one, the sums have 32 bits for that, and a weight's rounding to bf16 is relative.  With the exact maximum some row of a wave outgrows its own
// in most blocks, and every accumulator is multiplied for it.
constexpr float kTreeRaise = 6.0f;
constexpr int kTreeMaxNodes = 256;
constexpr int kTreeMaxWords = kTreeMaxNodes / 64;
constexpr int kTreeBlock = 16;                 // pages hold whole runs of this many keys
constexpr int kTreeMaxSplits = 64;

struct TreeArgs {
    const void *q, *k_cache, *v_cache;
    int64_t ldq;
    const int32_t *ctx, *row_start, *block_table;
    int64_t bt_stride;
    const uint64_t* mask;        // [tokens, words]; NULL: a chain (everything up to the node)
    int words;
    void* out;
    int64_t ldo;
    float *part, *state;         // splits: sums [split][token][head][d], (maximum, denominator) [split][token][head]
    int bt_cols, rows, tokens, max_nodes, hq, hkv, g, page, page_shift, num_pages, nsplit, row_blocks;
    int round_keys;              // keys that a split's workgroup takes in one round
    int row_part, slots, least;  // stacked rows of a workgroup, workgroups that run at once, rounds below which nothing is cut
    int per_unit;                // slots of a compute unit
    float scale_log2;
};

// Which keys and stacked rows a workgroup has: the grid is (8, row_blocks, places / 8), a place a row's split for one key/value head.  Workgroups go to the
// eight XCDs in turn, so the row_blocks workgroups that want the same keys are on one of them, and what one asks for the others find in its L2 (4 rows of
// 1200 keys, 64 nodes of 8B heads, 32 stacked rows a workgroup: 32 -> 21 us; where there are fewer places than XCDs x is 1).  Splits slowest: where
// no row is cut the first workgroups have the work.
struct TreePlace {
    int split, rb, kvh, b;
};
__device__ __forceinline__ TreePlace tree_place(const TreeArgs& a) {
    const unsigned place = blockIdx.z * gridDim.x + blockIdx.x, row = place / (unsigned)a.hkv, split = row / (unsigned)a.rows;
    unsigned b = row - split * a.rows;
    if (split > 0) b = (b + split) % (unsigned)a.rows;      // a row's splits on different XCDs (8 uneven rows, 48 nodes of one key/value head 37 -> 31 us)
    return {(int)split, (int)blockIdx.y, (int)(place - row * a.hkv), (int)b};
}

struct TreeSpan {
    int start, n, ctx, total;    // first token, nodes, cached tokens, keys that have a place in the table
};
__device__ __forceinline__ TreeSpan tree_span(const TreeArgs& a, int b) {
    TreeSpan s;      // (b is the same for a wave: scalar registers, whatever instruction loads them)
    s.start = min(max(__builtin_amdgcn_readfirstlane(a.row_start[b]), 0), a.tokens);
    s.n = min(min(max(__builtin_amdgcn_readfirstlane(a.row_start[b + 1]), s.start), a.tokens) - s.start, a.max_nodes);
    s.ctx = max(__builtin_amdgcn_readfirstlane(a.ctx[b]), 0);
    s.total = (int)min((int64_t)s.ctx + s.n, (int64_t)a.bt_cols << a.page_shift);
    return s;
}
// How many of the launch's splits a row of `total` keys takes.  A piece of work is a round (round_keys keys of up to row_part stacked rows of one
// key/value head); rows are cut so that no split has more than its share of the step's rounds over `slots` workgroups: where rows differ in
// length the long ones take more splits, and where there are rounds enough for every slot none is cut.  Nor is any where the longest row is no more than
// a compute unit's share of all (two workgroups run on one: 32 rows of 4096 to 8192 keys, 64 nodes of 8B heads, cut to their shares 265 us, whole 246).  In
// two halves, what a lane counts (its loads go out with a kernel's first) and their sums; all lanes of a wave call them together.
struct TreeWork {
    int rounds, longest;
};
__device__ __forceinline__ TreeWork step_work(const TreeArgs& a) {
    TreeWork w = {0, 0};
    if (a.nsplit > 1)
        for (int i = threadIdx.x & 63; i < a.rows; i += 64) {
            const int from = min(max(a.row_start[i], 0), a.tokens);
            const int n = min(min(max(a.row_start[i + 1], from), a.tokens) - from, a.max_nodes);
            const int keys = (int)min((int64_t)max(a.ctx[i], 0) + n, (int64_t)a.bt_cols << a.page_shift), rounds = (keys + a.round_keys - 1) / a.round_keys;
            w.rounds += (n * a.g + a.row_part - 1) / a.row_part * rounds;
            w.longest = max(w.longest, n > 0 ? rounds : 0);
        }
    return w;
}
template <int SHR> __device__ __forceinline__ void add_lanes(TreeWork& w) {      // from SHR lanes below, within rows of 16
    w.rounds += __builtin_amdgcn_update_dpp(0, w.rounds, 0x110 + SHR, 0xf, 0xf, true);
    w.longest = max(w.longest, __builtin_amdgcn_update_dpp(0, w.longest, 0x110 + SHR, 0xf, 0xf, true));
}
__device__ __forceinline__ int row_splits(const TreeArgs& a, int total, TreeWork w) {
    if (a.nsplit == 1) return 1;
    add_lanes<1>(w);
    add_lanes<2>(w);
    add_lanes<4>(w);
    add_lanes<8>(w);
    int64_t sum = 0;
    int longest = 0;
#pragma unroll
    for (int l = 15; l < 64; l += 16) {
        sum += __builtin_amdgcn_readlane(w.rounds, l);
        longest = max(longest, __builtin_amdgcn_readlane(w.longest, l));
    }
    const int share = max((int)((sum * a.hkv + a.slots - 1) / a.slots), a.least), rounds = (total + a.round_keys - 1) / a.round_keys;
    if (longest <= share * a.per_unit) return 1;
    return max(1, min(a.nsplit, (rounds + share - 1) / share));
}
// Which of the 32 keys from kb on a node sees (bit i: key kb + i): cached tokens all, nodes by its mask, whose first word is given
__device__ __forceinline__ uint32_t visible_keys(const TreeArgs& a, const TreeSpan& s, int node, uint64_t word0, int kb) {
    const int first = kb - s.ctx;
    if (!a.mask) {
        const int up = node + 1 - first;
        return up >= 32 ? ~0u : up > 0 ? (1u << up) - 1 : 0;
    }
    if (first < 0) return first <= -32 ? ~0u : (uint32_t)(word0 << -first) | ((1u << -first) - 1);
    const int at = first >> 6, sh = first & 63;
    const uint64_t* w = a.mask + (int64_t)(s.start + node) * a.words;
    uint64_t v = (at == 0 ? word0 : at < a.words ? w[at] : 0) >> sh;
    if (sh > 32 && at + 1 < a.words) v |= w[at + 1] << (64 - sh);
    return (uint32_t)v;
}

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(4))) short s16x4_t;

__device__ __forceinline__ float max_of_quarters(float v) {      // over lanes l, l ^ 16, l ^ 32, l ^ 48, in the vector unit
    const unsigned u = __float_as_uint(v);
    const auto x = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const float m = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
    const unsigned w = __float_as_uint(m);
    const auto y = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
}
// infinities and NaN of two packed bf16 become zero; whether there were any
__device__ __forceinline__ bool drop_odd(uint32_t& w) {
    const bool lo = (w & 0x7f80u) == 0x7f80u, hi = (w & 0x7f800000u) == 0x7f800000u;
    w &= (lo ? 0xffff0000u : ~0u) & (hi ? 0x0000ffffu : ~0u);
    return lo || hi;
}

template <bool F32> struct TreeT;
template <> struct TreeT<true> {
    typedef float T;
    static __device__ __forceinline__ f32x4_t ld4(const float* p) { return *reinterpret_cast<const f32x4_t*>(p); }
    static __device__ __forceinline__ void st4(float* p, f32x4_t v) { *reinterpret_cast<f32x4_t*>(p) = v; }
};
template <> struct TreeT<false> {
    typedef uint16_t T;
    static __device__ __forceinline__ f32x4_t ld4(const uint16_t* p) {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        return (f32x4_t){bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y)};
    }
    static __device__ __forceinline__ void st4(uint16_t* p, f32x4_t v) {
        *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    }
};

// dimensions c .. c + 3 of a stacked row: the output, or a split's sums
template <bool F32, int D>
__device__ __forceinline__ void leave_rows(const TreeArgs& a, const TreeSpan& s, bool whole, int split, int kvh, int sr, int c, float top,
                                           float den, f32x4_t o) {
    typedef TreeT<F32> X;
    const int64_t t = s.start + sr / a.g;
    const int head = kvh * a.g + sr % a.g;
    if (whole) {
        const float inv = den != 0.f ? 1.0f / den : 0.f;      // nothing visible: zeros
        X::st4((typename X::T*)a.out + t * a.ldo + (int64_t)head * D + c, o * inv);
    } else {
        const int64_t at = ((int64_t)split * a.tokens + t) * a.hq + head;
        *reinterpret_cast<f32x4_t*>(a.part + at * D + c) = o;
        if (c == 0) {
            a.state[2 * at] = top;
            a.state[2 * at + 1] = den;
        }
    }
}

// Values that are not finite, of keys that some row may not see, are left out of a split's products; here they are handed, key by key, to
// the sums of a row that sees them: whatever its weight, the result is that infinity or NaN.  The keys: runs of `span` from `first` on, `step`
// apart, up to `end`; `block` is how many the kernel takes together (one with nothing to hide went through the product whole).  Rare, and slow.
template <bool F32, int D, class Take>
__device__ __forceinline__ void odd_values(const TreeArgs& a, const TreeSpan& s, int b, int kvh, int node, int first, int step, int span,
                                           int end, int block, Take&& take) {
    const int32_t* bt = a.block_table + (int64_t)b * a.bt_stride;
    for (; first < end; first = step > end - first ? end : first + step)
        for (int key = first; key < min(first + span, end); ++key) {
            const int pg = bt[key >> a.page_shift], kb = key / block * block;
            if (pg < 0 || pg >= a.num_pages) continue;
            if (kb + block <= s.ctx && kb + block <= s.total) {
                bool there = true;
                for (int k = kb; k < kb + block; k += kTreeBlock) there &= (unsigned)bt[k >> a.page_shift] < (unsigned)a.num_pages;
                if (there) continue;
            }
            const int j = key - s.ctx;
            if (j >= 0 && (a.mask ? !(a.mask[(int64_t)(s.start + node) * a.words + (j >> 6)] >> (j & 63) & 1) : j > node)) continue;
            take((const typename TreeT<F32>::T*)a.v_cache + ((((int64_t)pg << a.page_shift) + (key & (a.page - 1))) * a.hkv + kvh) * D);
        }
}
__device__ __forceinline__ bool is_odd(float x) { return !(fabsf(x) <= 3.4028235e38f); }
// dimensions c .. c + 3 of a stacked row, of a kernel that deals its blocks
template <bool F32, int D>
__device__ __forceinline__ void add_odd(const TreeArgs& a, const TreeSpan& s, int b, int kvh, int split, int splits, int block, int sr, int c,
                                        f32x4_t& o) {
    odd_values<F32, D>(a, s, b, kvh, sr / a.g, split * a.round_keys, splits * a.round_keys, a.round_keys, s.total, block,
                       [&](const typename TreeT<F32>::T* v) {
                           const f32x4_t x = TreeT<F32>::ld4(v + c);
#pragma unroll
                           for (int j = 0; j < 4; ++j)
                               if (is_odd(x[j])) o[j] += x[j];
                       });
}

// ------------------------------------------------------------------ fp32
// Both products on v_mfma_f32_16x16x4_f32 (operand A lane (r, q) = A[r][slot q], B likewise, result lane (r, q) = C[4 q + j][r]); the
// contraction's slots are labels.  S^T = K . Q^T: slot q of step j of a group of 16 dimensions is dimension 4 q + j, so a key's and a
// query's values are read 16 (8) bytes a lane.  O^T = V^T . P^T: slot q of step j is key 4 q + j, which is where S^T left its score;
// row r of output block c is dimension 64 h + 4 r + c, so a value row too is read as it lies.  Nothing goes through LDS until the end.  The
// next block's keys are requested into the registers that the scores leave, its values into those that the sums leave.
template <int D, int RT>
__global__ __launch_bounds__(256, 2) void tree_attn_f32_kernel(TreeArgs a) {
    constexpr bool F32 = true;
    constexpr int W = 4, KG = D / 16, H = D / 64;
    __shared__ __attribute__((aligned(16))) float oL[W][RT * 16][D + 4];
    __shared__ float mL[W][RT * 16], lL[W][RT * 16];
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
    const TreePlace w = tree_place(a);
    const int split = w.split, rb = w.rb, kvh = w.kvh, b = w.b;
    if (split >= a.nsplit) return;
    typedef const int32_t __attribute__((address_space(4))) Entry;      // (nothing here writes the table: scalar loads)
    Entry* bt = (Entry*)(uintptr_t)(a.block_table + (int64_t)b * a.bt_stride);
    auto page_of = [&](int blk) { return bt[min((blk * kTreeBlock) >> a.page_shift, a.bt_cols - 1)]; };
    int blk = split * W + wid, pg = page_of(blk);
    const TreeWork work = step_work(a);
    const TreeSpan s = tree_span(a, b);
    const int stacked = s.n * a.g, row0 = rb * RT * 16;
    const int blocks = (s.total + kTreeBlock - 1) / kTreeBlock;
    if (row0 >= stacked || (split > 0 && split * a.round_keys >= s.total)) return;
    const int splits = row_splits(a, s.total, work);
    if (split >= splits) return;

    const unsigned row_bytes = (unsigned)a.hkv * D * 4, k_at = r * row_bytes + 16 * q, v_at = 4 * q * row_bytes + 16 * r;
    auto base_of = [&](const void* cache, int at, int page) {
        const int64_t row = ((int64_t)(page >= 0 && page < a.num_pages ? page : 0) << a.page_shift) + ((at * kTreeBlock) & (a.page - 1));
        return (const unsigned char*)cache + row * row_bytes + kvh * D * 4;
    };
    f32x4_t kf[KG], vf[4][H];
    auto load_k = [&](int at, int page) {
        const unsigned char* p = base_of(a.k_cache, at, page);
#pragma unroll
        for (int k = 0; k < KG; ++k) kf[k] = *reinterpret_cast<const f32x4_t*>(p + 64 * k + k_at);
    };
    auto load_v = [&](int at, int page) {
        const unsigned char* p = base_of(a.v_cache, at, page);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int h = 0; h < H; ++h) vf[j][h] = *reinterpret_cast<const f32x4_t*>(p + j * row_bytes + 256 * h + v_at);
    };
    load_k(blk, pg);
    load_v(blk, pg);

    f32x4_t qf[RT][KG];
    int node[RT];
    uint64_t word0[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int sr = min(row0 + i * 16 + r, stacked - 1);
        node[i] = sr / a.g;
        const float* qp = (const float*)a.q + (int64_t)(s.start + node[i]) * a.ldq + (int64_t)(kvh * a.g + sr % a.g) * D + 4 * q;
#pragma unroll
        for (int k = 0; k < KG; ++k) qf[i][k] = *reinterpret_cast<const f32x4_t*>(qp + 16 * k);
        word0[i] = a.mask ? a.mask[(int64_t)(s.start + node[i]) * a.words] : 0;
    }
    f32x4_t acc[RT][H][4];
    float m[RT], l[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        m[i] = kTreeNegBig;
        l[i] = 0.f;
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[i][h][c] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    }
    bool odd = false;
    while (blk < blocks) {
        const int kb = blk * kTreeBlock, next = blk + splits * W, left = s.total - kb;
        const uint32_t valid = pg < 0 || pg >= a.num_pages ? 0 : left < 16 ? (1u << left) - 1 : 0xffffu;
        const bool open = valid == 0xffffu && kb + kTreeBlock <= s.ctx;      // every key there and visible to every row (uniform)
        const int pn = next < blocks ? page_of(next) : -1;
        f32x4_t sc[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) sc[i] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KG; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < RT; ++i) sc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[k][j], qf[i][k][j], sc[i], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        if (next < blocks) load_k(next, pn);
        __builtin_amdgcn_sched_barrier(0);
        f32x4_t p[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            if (!open) {
                const uint32_t seen = visible_keys(a, s, node[i], word0[i], kb) & valid;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (!(seen >> (4 * q + j) & 1)) sc[i][j] = -__builtin_inff();
            }
            const float top = max_of_quarters(fmaxf(fmaxf(sc[i][0], sc[i][1]), fmaxf(sc[i][2], sc[i][3])) * a.scale_log2);
            if (__builtin_amdgcn_ballot_w64(top > m[i] + kTreeRaise) != 0) {
                const float mn = fmaxf(m[i], top), alpha = __builtin_amdgcn_exp2f(m[i] - mn);
                m[i] = mn;
                l[i] *= alpha;
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[i][h][c] *= alpha;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) p[i][j] = __builtin_amdgcn_exp2f(fmaf(sc[i][j], a.scale_log2, -m[i]));
            l[i] += (p[i][0] + p[i][1]) + (p[i][2] + p[i][3]);
        }
        // Where a row may not see a key, its weight is zero and the product would still hand on a value that is not finite: such
        // values are left out here and added at the end (add_odd); of keys that do not count everything is left out.
        if (!open) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        if (!(valid >> (4 * q + j) & 1)) vf[j][h][c] = 0.f;
                        if (is_odd(vf[j][h][c])) {
                            vf[j][h][c] = 0.f;
                            odd = true;
                        }
                    }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int i = 0; i < RT; ++i)
                        acc[i][h][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[j][h][c], p[i][j], acc[i][h][c], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        if (next < blocks) load_v(next, pn);
        __builtin_amdgcn_sched_barrier(0);
        blk = next;
        pg = pn;
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        l[i] += __shfl_xor(l[i], 16, 64);
        l[i] += __shfl_xor(l[i], 32, 64);
        if (q == 0) {
            mL[wid][i * 16 + r] = m[i];
            lL[wid][i * 16 + r] = l[i];
        }
        // lane (r, q): dimensions 64 h + 16 q + 4 e + c of stacked row r
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                *reinterpret_cast<f32x4_t*>(&oL[wid][i * 16 + r][64 * h + 16 * q + 4 * e]) =
                    (f32x4_t){acc[i][h][0][e], acc[i][h][1][e], acc[i][h][2][e], acc[i][h][3][e]};
    }
    const bool any_odd = __syncthreads_or(odd);
    const bool whole = splits == 1;
#pragma unroll 1
    for (int it = threadIdx.x; it < RT * 16 * (D / 4); it += 256) {
        const int rr = it / (D / 4), c = it % (D / 4) * 4, sr = row0 + rr;
        if (sr >= stacked) break;
        float top = mL[0][rr];
#pragma unroll
        for (int w = 1; w < W; ++w) top = fmaxf(top, mL[w][rr]);
        float den = 0.f;
        f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float f = __builtin_amdgcn_exp2f(mL[w][rr] - top);
            den = fmaf(lL[w][rr], f, den);
            o += *reinterpret_cast<const f32x4_t*>(&oL[w][rr][c]) * f;
        }
        if (any_odd) add_odd<F32, D>(a, s, b, kvh, split, splits, 16, sr, c, o);
        leave_rows<F32, D>(a, s, whole, split, kvh, sr, c, top, den, o);
    }
}

// ------------------------------------------------------------------ bf16, up to 64 stacked rows (heads of 128: 32)
// Each of W waves has keys of its own (32 at a time) and all the rows: nothing is shared until the end, no barrier in the loop.
//   S^T = K . Q^T   v_mfma_f32_16x16x32_bf16, operand A = key rows as they lie in memory (lane (r, q): row r, dimensions 32 k + 8 q ..);
//   O^T = V^T . P^T operand B = P as S^T left it, rounded to bf16 (keys 4 q + j and 16 + 4 q + j), operand A through the wave's own piece of
//                   LDS with the transposing read, which delivers those keys.
// The normaliser sums the unrounded weights; rounding a weight to bf16 (2^-8 of it) is what the matrix instruction asks for: results are
// 2.0 to 2.3e-3 of their size off 64 bits, where weights in 32 bits give 1.65e-3, the output's rounding alone.  The next block's keys and values are
// requested into the registers that this one leaves.
// Keys as the operand wants them are sixteen rows a quarter wave, which a compute unit's address path serves at a third of the rate of whole rows;
// for 16 rows of heads of 128, where registers allow, they are read row by row and turned in LDS as well, and the next block's requests go out in front
// of the first product: 8 heads of 128 on 1, 7 nodes, 45 keys 7.5 -> 6.4 us, 900 in one piece 15.6 -> 13.7.  (Heads of 64 are a piece's latency
// slower for it, 900 keys 9.1 -> 10.0; with 32 rows registers spill.)
template <int D, int RT>
constexpr bool kNarrowTurn = D == 128 && RT == 1;
template <int D, int RT, int W>
constexpr size_t kNarrowLds = [] {
    constexpr size_t stage = W * 32 * (D * 2 + 32 + (kNarrowTurn<D, RT> ? D * 2 : 0)), merge = W * RT * 16 * (D + 4) * sizeof(float);
    return stage > merge ? stage : merge;
}();

template <int D, int RT, int W>
__global__ __launch_bounds__(W * 64, 2) void tree_attn_narrow_kernel(TreeArgs a) {
    constexpr int KS = D / 32, DT = D / 16, RB = D * 2, VROW = RB + 32, VPR = D / 8, NV = 32 * VPR / 64, OROW = D + 4, ROWS = RT * 16;
    constexpr bool TURN = kNarrowTurn<D, RT>;
    static_assert(NV == 2 * KS, "a block's keys are as many pieces either way");
    __shared__ __attribute__((aligned(16))) unsigned char lds[kNarrowLds<D, RT, W>];
    __shared__ float mL[W][ROWS], lL[W][ROWS];
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
    const TreePlace w = tree_place(a);
    const int split = w.split, rb = w.rb, kvh = w.kvh, b = w.b;
    if (split >= a.nsplit) return;
    typedef const int32_t __attribute__((address_space(4))) Entry;      // (nothing here writes the table: scalar loads)
    Entry* bt = (Entry*)(uintptr_t)(a.block_table + (int64_t)b * a.bt_stride);
    auto pages_of = [&](int blk, int (&pg)[2]) {
        pg[0] = bt[min((blk * 32) >> a.page_shift, a.bt_cols - 1)];
        pg[1] = bt[min((blk * 32 + 16) >> a.page_shift, a.bt_cols - 1)];
    };
    int blk = split * W + wid, pg[2];
    bool odd = false;
    pages_of(blk, pg);
    const TreeWork work = step_work(a);
    const TreeSpan s = tree_span(a, b);
    const int stacked = s.n * a.g, row0 = rb * ROWS, blocks = (s.total + 31) / 32;
    if (row0 >= stacked || (split > 0 && split * a.round_keys >= s.total)) return;
    const int splits = row_splits(a, s.total, work);
    if (split >= splits) return;

    // (a request = a base that is the same for the wave, in scalar registers, and a lane's offset of 32 bits that never changes)
    const unsigned row_bytes = (unsigned)a.hkv * D * 2, k_at = r * row_bytes + 16 * q, v_from = (lane / VPR) * row_bytes + (lane % VPR) * 16;
    uint4 kR[NV], vR[NV];
    auto base_of = [&](const void* cache, int at, int half, int page) {
        const int64_t row = ((int64_t)(page >= 0 && page < a.num_pages ? page : 0) << a.page_shift) + ((at * 32 + 16 * half) & (a.page - 1));
        return (const unsigned char*)cache + row * row_bytes + kvh * RB;
    };
    auto load_rows = [&](const void* cache, int at, const int (&page)[2], uint4 (&to)[NV]) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const unsigned char* p = base_of(cache, at, x, page[x]);
#pragma unroll
            for (int i = 0; i < NV / 2; ++i) to[x * (NV / 2) + i] = ld16(p + i * (64 / VPR) * row_bytes + v_from);
        }
    };
    auto load_k = [&](int at, const int (&page)[2]) {
        if constexpr (TURN) {
            load_rows(a.k_cache, at, page, kR);
        } else {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const unsigned char* p = base_of(a.k_cache, at, x, page[x]);
#pragma unroll
                for (int k = 0; k < KS; ++k) kR[x * KS + k] = ld16(p + 64 * k + k_at);
            }
        }
    };
    load_k(blk, pg);
    load_rows(a.v_cache, blk, pg, vR);
    int pn[2] = {-1, -1};      // pages of the next block
    if (blk + splits * W < blocks) pages_of(blk + splits * W, pn);

    bf16x8_t qf[RT][KS];
    int node[RT];
    uint64_t word0[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int sr = min(row0 + i * 16 + r, stacked - 1);
        node[i] = sr / a.g;
        const uint16_t* qp = (const uint16_t*)a.q + (int64_t)(s.start + node[i]) * a.ldq + (int64_t)(kvh * a.g + sr % a.g) * D + 8 * q;
#pragma unroll
        for (int k = 0; k < KS; ++k) qf[i][k] = __builtin_bit_cast(bf16x8_t, ld16(qp + 32 * k));
        word0[i] = a.mask ? a.mask[(int64_t)(s.start + node[i]) * a.words] : 0;
    }
    f32x4_t acc[RT][DT];
    float m[RT], l[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        m[i] = kTreeNegBig;
        l[i] = 0.f;
#pragma unroll
        for (int t = 0; t < DT; ++t) acc[i][t] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    }
    unsigned char *vst = lds + wid * (32 * (VROW + (TURN ? RB : 0))), *kst = vst + 32 * VROW;
    // (the image of the keys is their rows back to back, 16-byte piece c of row r at c ^ (r % 16): sixteen rows' pieces lie in sixteen banks' places)
    const int k_to = (lane / VPR) * RB, k_col = ((lane % VPR) ^ q) * 16, k_row = r * RB, k_piece = (q ^ r) * 16;
    const int v_at = (lane / VPR) * VROW + (lane % VPR) * 16, tr_at = (4 * q + (r >> 2)) * VROW + (r & 3) * 8;

    while (blk < blocks) {
        const int kb = blk * 32, next = blk + splits * W;
        uint32_t valid = (pg[0] >= 0 && pg[0] < a.num_pages ? 0xffffu : 0) | (pg[1] >= 0 && pg[1] < a.num_pages ? 0xffff0000u : 0);
        if (s.total - kb < 32) valid &= (1u << (s.total - kb)) - 1;
        const bool open = valid == ~0u && kb + 32 <= s.ctx;       // every key there and visible to every row (uniform)
        if (!open) {     // values of keys that do not count are zero, what is not finite is added at the end (add_odd)
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const bool there = valid >> (i * (64 / VPR) + lane / VPR) & 1;
                if (!there) vR[i] = make_uint4(0, 0, 0, 0);
                const bool o0 = drop_odd(vR[i].x), o1 = drop_odd(vR[i].y), o2 = drop_odd(vR[i].z), o3 = drop_odd(vR[i].w);
                odd |= o0 | o1 | o2 | o3;
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if constexpr (TURN) *reinterpret_cast<uint4*>(kst + k_to + i * (64 / VPR) * RB + (k_col ^ (64 * (i % (NV / 2))))) = kR[i];
            *reinterpret_cast<uint4*>(vst + v_at + i * (64 / VPR) * VROW) = vR[i];
        }
        auto request = [&] {      // (the requests go into registers that LDS writes, or the products, have read: not before them)
            __builtin_amdgcn_sched_barrier(0);
            if (next < blocks) {
                load_k(next, pn);
                load_rows(a.v_cache, next, pn, vR);
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        bf16x8_t kf[2][KS];
        if constexpr (TURN) request();
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int k = 0; k < KS; ++k)
                kf[x][k] = __builtin_bit_cast(bf16x8_t, TURN ? *reinterpret_cast<const uint4*>(kst + k_row + 16 * x * RB + (k_piece ^ (64 * k))) : kR[x * KS + k]);
        f32x4_t sc[RT][2];
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                sc[i][x] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < KS; ++k)
                    sc[i][x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[x][k], qf[i][k], sc[i][x], 0, 0, 0);
            }
        if constexpr (!TURN) request();
        pg[0] = pn[0];
        pg[1] = pn[1];
        pn[0] = pn[1] = -1;
        if (next + splits * W < blocks) pages_of(next + splits * W, pn);
        bf16x8_t pf[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            if (!open) {
                const uint32_t seen = visible_keys(a, s, node[i], word0[i], kb) & valid;
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (!(seen >> (16 * x + 4 * q + j) & 1)) sc[i][x][j] = -__builtin_inff();
            }
            float top = fmaxf(fmaxf(fmaxf(sc[i][0][0], sc[i][0][1]), fmaxf(sc[i][0][2], sc[i][0][3])),
                              fmaxf(fmaxf(sc[i][1][0], sc[i][1][1]), fmaxf(sc[i][1][2], sc[i][1][3]))) * a.scale_log2;
            top = max_of_quarters(top);
            if (__builtin_amdgcn_ballot_w64(top > m[i] + kTreeRaise) != 0) {
                const float mn = fmaxf(m[i], top), alpha = __builtin_amdgcn_exp2f(m[i] - mn);
                m[i] = mn;
                l[i] *= alpha;
#pragma unroll
                for (int t = 0; t < DT; ++t) acc[i][t] *= alpha;
            }
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(sc[i][e >> 2][e & 3], a.scale_log2, -m[i]));
            l[i] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
            pf[i] = __builtin_bit_cast(bf16x8_t, make_uint4(pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]), pack_bf16x2(p[4], p[5]),
                                                            pack_bf16x2(p[6], p[7])));
        }
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            const unsigned char* vb = vst + tr_at + 32 * t;
            const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4_t __attribute__((address_space(3)))*)(vb));
            const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4_t __attribute__((address_space(3)))*)(vb + 16 * VROW));
            const s16x8_t both = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
            for (int i = 0; i < RT; ++i)
                acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, both), pf[i], acc[i][t], 0, 0, 0);
        }
        blk = next;
    }
    __syncthreads();       // (the states lie where values were staged)
    float* oL = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        l[i] += __shfl_xor(l[i], 16, 64);
        l[i] += __shfl_xor(l[i], 32, 64);
        if (q == 0) {
            mL[wid][i * 16 + r] = m[i];
            lL[wid][i * 16 + r] = l[i];
        }
#pragma unroll
        for (int t = 0; t < DT; ++t) *reinterpret_cast<f32x4_t*>(oL + (wid * ROWS + i * 16 + r) * OROW + 16 * t + 4 * q) = acc[i][t];
    }
    const bool any_odd = __syncthreads_or(odd);
    const bool whole = splits == 1;
#pragma unroll 1
    for (int it = threadIdx.x; it < ROWS * (D / 4); it += W * 64) {
        const int rr = it / (D / 4), c = it % (D / 4) * 4, sr = row0 + rr;
        if (sr >= stacked) break;
        float top = mL[0][rr];
#pragma unroll
        for (int w = 1; w < W; ++w) top = fmaxf(top, mL[w][rr]);
        float den = 0.f;
        f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float f = __builtin_amdgcn_exp2f(mL[w][rr] - top);
            den = fmaf(lL[w][rr], f, den);
            o += *reinterpret_cast<const f32x4_t*>(oL + (w * ROWS + rr) * OROW + c) * f;
        }
        if (any_odd) add_odd<false, D>(a, s, b, kvh, split, splits, 32, sr, c, o);
        leave_rows<false, D>(a, s, whole, split, kvh, sr, c, top, den, o);
    }
}

// ------------------------------------------------------------------ bf16, more rows: 32 a wave, keys shared by the workgroup
// 128 stacked rows against every 64-key tile in LDS, one barrier a tile, two workgroups a compute unit (two waves a SIMD that do not wait for each
// other's barriers, and shorter trees leave less idle than in one of 256 rows).  Keys and values go to LDS by global_load_lds, KD - 1 and VD tiles'
// time ahead (no staging registers).
//   * v_mfma_f32_32x32x16_bf16: S^T = K . Q^T leaves a lane (row l & 31, half h = l >> 5) 16 scores of a 32-key block, keys (i & 3) + 8 (i >> 2) +
//     4 h; registers 8 s .. 8 s + 7, rounded to bf16, are operand B of step s of O^T += V^T . P^T as they stand, and the transposing reads of
//     V deliver those keys.
//   * pipeline over 32-key blocks: the matrix unit forms S of block u + 1 and adds V^T P of u, the vector unit turns scores into weights, half of a
//     block's in the step behind their product and half in the next, LDS reads run a few matrix instructions ahead, requests go out one a slot.  All of
//     it is dealt out slot by slot (a matrix instruction each) between scheduling fences.  A tile takes 0.8 us where 0.43 are matrix instructions (1.05 with
//     a block's weights all in one step, all requests in front and a scalar page number a tile).
//   * no running maximum: weights are 2^(s - m) with m the maximum of the row's first block.  Their size does not touch their precision (bf16 and
//     the fp32 sums are relative), only their range, so a row whose denominator or sums leave the range that is safe - scores 44 nats above those of
//     its first block - makes the workgroup do its keys again with a running maximum.  (The maximum of every block, its exchange between lanes and
//     the test for a rescale were a fifth of the vector unit's work: 32 rows of 4096 and 64 nodes 188 -> 165 us, now 151.)
//   * a tile in which every key counts for every row (all but the one or two with nodes in them) takes no mask; the others, and the second pass, go through
//     a plainer step.
// Waves without rows (short trees) only stage.  KW 2, for up to 64 rows: two waves take the two 32-key blocks of a tile for the same 32 rows and join
// their states at the end.
typedef __attribute__((ext_vector_type(16))) float f32x16_t;

__device__ __forceinline__ float max3_tree(float a, float b, float c) {      // (fmaxf of a product's result is a self-maximum more)
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// all but the youngest N requests have landed
template <int N>
__device__ __forceinline__ void wait_landed() {
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

template <int D, int KW, int KD>
__global__ __launch_bounds__(256, 2) void tree_attn_wide_kernel(TreeArgs a) {
    constexpr int KT = 64, KS = D / 16, DB = D / 32, NP = 2 * DB;
    constexpr int PF = 3, PFV = NP - 1 < 7 ? NP - 1 : 7;        // reads of keys and values in front of their matrix instruction
    constexpr int VD = KD - 1, RB = D * 2, TB = KT * RB, VPR = D / 8, NI = TB / 4096;      // NI: requests of a wave for a tile
    __shared__ __attribute__((aligned(16))) unsigned char ring[(KD + 1 + VD + 1) * TB];
    unsigned char *const kring = ring, *const vring = ring + (KD + 1) * TB;
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lq = lane & 31, hi = lane >> 5;

    const TreePlace w = tree_place(a);
    const int split = w.split, rb = w.rb, kvh = w.kvh, b = w.b;
    if (split >= a.nsplit) return;
    const TreeWork work = step_work(a);
    const TreeSpan s = tree_span(a, b);
    // a row's stacked rows in as few parts as 128 (64) allow, of even size
    const int stacked = s.n * a.g, parts = (stacked + 128 / KW - 1) / (128 / KW);
    if (rb >= parts || (split > 0 && split * 64 * a.least >= s.total)) return;
    const int splits = row_splits(a, s.total, work);
    if (split >= splits) return;
    const int part_rows = ((stacked + parts - 1) / parts + 31) & ~31, row0 = rb * part_rows;
    if (row0 >= stacked) return;
    const int tiles = (s.total + KT - 1) / KT, per = (tiles + splits - 1) / splits, t0 = split * per, t1 = min(t0 + per, tiles);
    const int my_rows = min(part_rows, stacked - row0);
    const int rg = KW == 1 ? wid : wid & 1, kh = KW == 1 ? 0 : wid >> 1;      // the wave's rows, and its block of a tile
    const bool active = rg * 32 < my_rows;                      // uniform over the wave
    const int sr = min(row0 + rg * 32 + lq, stacked - 1), node = sr / a.g, head = kvh * a.g + sr - node * a.g;
    const bool stored = rg * 32 + lq < my_rows;

    bf16x8_t qf[KS];
    {
        const uint16_t* qp = (const uint16_t*)a.q + (int64_t)(s.start + node) * a.ldq + (int64_t)head * D + hi * 8;
#pragma unroll
        for (int k = 0; k < KS; ++k) qf[k] = __builtin_bit_cast(bf16x8_t, ld16(qp + k * 16));
    }
    // ---- pages: the four runs of 16 keys of a tile lie in a page each; a wave stages one of them.  The numbers of 64 tiles are asked for at once: lane l has
    // the page of the wave's run of tile tb + l, and which of that tile's four runs have one (a scalar load a tile, waited for with every LDS read on
    // its way, was a tenth of the loop)
    const int32_t* table = a.block_table + (int64_t)b * a.bt_stride;
    int tb, ids, oks, open_end;      // open_end: tiles in front of this one take no mask, as far as their pages are known
    auto fill = [&](int t) __attribute__((always_inline)) {
        tb = t;
        const int kb = min(t + lane, t1 - 1) * KT;
        ids = table[min((kb + 16 * wid) >> a.page_shift, a.bt_cols - 1)];
        oks = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) oks |= (int)((unsigned)table[min((kb + 16 * i) >> a.page_shift, a.bt_cols - 1)] < (unsigned)a.num_pages) << i;
        asm volatile("" : "+v"(ids));      // (both have landed: nothing waits for them in the loop)
        const uint64_t holes = __builtin_amdgcn_ballot_w64(oks != 15);
        if (holes) open_end = min(open_end, t + __builtin_ctzll(holes));
    };
    auto counted = [&](int t) __attribute__((always_inline)) -> uint64_t {      // keys of a tile that count (the last splits may have no tile)
        const int left = s.total - t * KT, ok = __builtin_amdgcn_readlane(oks, min(t, t1 - 1) - tb);
        uint64_t there = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) there |= ok >> i & 1 ? 0xffffull << (16 * i) : 0;
        return left < KT ? there & ((1ull << max(left, 0)) - 1) : there;
    };
    auto open_tile = [&](int t, uint64_t bits) __attribute__((always_inline)) { return bits == ~0ull && (t + 1) * KT <= s.ctx; };
    const unsigned row_bytes = (unsigned)a.hkv * RB;
    auto base_of = [&](int t) __attribute__((always_inline)) {      // byte offset in either cache of the wave's first row
        const int at = min(t, t1 - 1), page = __builtin_amdgcn_readlane(ids, at - tb);
        const int64_t row = ((int64_t)((unsigned)page < (unsigned)a.num_pages ? page : 0) << a.page_shift) + ((at * KT + 16 * wid) & (a.page - 1));
        return row * row_bytes + kvh * RB;
    };
    // The LDS image of a tile is its rows back to back; 16-byte piece c of row r stands at c ^ k_turn(r) (keys: operand reads of 16 rows) or
    // c ^ v_turn(r) (values: transposing reads of four pieces of four rows), which keeps the reads free of bank conflicts.  A request of a
    // wave is a KB of the image; the lanes ask for the pieces that belong there.
    auto k_turn = [](int r) __attribute__((always_inline)) { return D == 128 ? r & 15 : (r >> 1) & 7; };
    auto v_turn = [](int r) __attribute__((always_inline)) { return D == 128 ? (r & 3) << 2 : (r >> 1 & 1) << 2; };
    unsigned k_from[NI], v_from[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int r = i * (64 / VPR) + lane / VPR, c = lane % VPR;      // (a run's first row turns nothing: r for 16 wid + r)
        k_from[i] = r * row_bytes + (c ^ k_turn(r)) * 16;
        v_from[i] = r * row_bytes + (c ^ v_turn(r)) * 16;
    }
    // (through inline assembly: seen by the compiler, these loads make it wait for all of them in front of every LDS read)
    auto copy = [&](const void* cache, int64_t base, unsigned from, const unsigned char* to) __attribute__((always_inline)) {
        const unsigned dst = (unsigned)(size_t)(__attribute__((address_space(3))) const unsigned char*)to;
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                     : : "v"(from), "s"((const unsigned char*)cache + base), "s"(dst) : "memory");
    };
    auto copy_k = [&](int64_t base, int slot, int i) __attribute__((always_inline)) {
        copy(a.k_cache, base, k_from[i], kring + slot * TB + wid * 16 * RB + i * 1024);
    };
    auto copy_v = [&](int64_t base, int slot, int i) __attribute__((always_inline)) {
        copy(a.v_cache, base, v_from[i], vring + slot * TB + wid * 16 * RB + i * 1024);
    };
    // values of keys that do not count become zero, and what is not finite of the others is left for the end: in the pieces that this wave asked
    // for, once they are there
    bool odd = false;
    auto clean = [&](int slot, uint64_t bits) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            uint4* at = reinterpret_cast<uint4*>(vring + slot * TB + wid * 16 * RB + i * 1024 + lane * 16);
            uint4 v = *at;
            if (!(bits >> (16 * wid + i * (64 / VPR) + lane / VPR) & 1)) v = make_uint4(0, 0, 0, 0);
            const bool o0 = drop_odd(v.x), o1 = drop_odd(v.y), o2 = drop_odd(v.z), o3 = drop_odd(v.w);
            odd |= o0 | o1 | o2 | o3;
            *at = v;
        }
    };
    // which of a tile's keys the lane's row sees
    auto visible = [&](int t, uint64_t bits) __attribute__((always_inline)) -> uint64_t {
        const int first = t * KT - s.ctx;
        if (first <= -KT) return bits;
        if (!a.mask) {
            const int up = node + 1 - first;
            return bits & (up >= 64 ? ~0ull : (1ull << max(up, 0)) - 1);
        }
        const uint64_t* w = a.mask + (int64_t)(s.start + node) * a.words;
        if (first < 0) return bits & ((w[0] << -first) | ((1ull << -first) - 1));
        const int at = first >> 6, sh = first & 63;
        uint64_t v = at < a.words ? w[at] >> sh : 0;
        if (sh && at + 1 < a.words) v |= w[at + 1] << (64 - sh);
        return bits & v;
    };

    // ---- fragments
    const int li = lane & 15, v_row = 4 * hi + (li >> 2);
    const unsigned k_at = lq * RB + ((hi ^ k_turn(lq)) * 16);
    const unsigned v_at = v_row * RB + ((2 * ((lane >> 4) & 1) + ((li & 3) >> 1)) ^ v_turn(v_row)) * 16 + (li & 1) * 8;
    auto k_frag = [&](const unsigned char* kblock, int k) __attribute__((always_inline)) {
        return __builtin_bit_cast(bf16x8_t, *reinterpret_cast<const uint4*>(kblock + (k_at ^ (32 * k))));
    };
    auto v_frag = [&](const unsigned char* vblock, int j) __attribute__((always_inline)) {      // step j / DB, rows 32 (j % DB) of O^T
        const unsigned char* vb = vblock + (j / DB) * 16 * RB + (v_at ^ (64 * (j % DB)));
        const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4_t __attribute__((address_space(3)))*)(vb));
        const s16x4_t up = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4_t __attribute__((address_space(3)))*)(vb + 8 * RB));
        const s16x8_t both = {lo[0], lo[1], lo[2], lo[3], up[0], up[1], up[2], up[3]};
        return __builtin_bit_cast(bf16x8_t, both);
    };

    f32x16_t oacc[DB];
    float mrun = kTreeNegBig, lrun0 = 0.f, lrun1 = 0.f;
    bool saw = false;                  // any key
    uint32_t pw[8];
    float fa[8][2], eb[8][2];
    // The eight pairs of a lane's scores of a block take three stages, a slot apart: product with the scale, exponential, sum and packing.  A block's slots are
    // numbered from the step that adds its values; the first pairs go through during the step before (negative numbers), behind that step's scores, so
    // that the vector unit has about as much to do in every slot.  Pairs 0 to 3 are due in slot KS, 4 to 7 in KS + DB.
    constexpr int NS = KS + NP;
    auto softmax_slot = [&](const f32x16_t& sc, int at) __attribute__((always_inline)) {
        constexpr int kEnter128[8] = {-5, -3, 0, 2, 4, 6, 8, 9}, kEnter64[8] = {-3, -2, -1, 0, 0, 1, 2, 3};
#pragma unroll
        for (int pr = 0; pr < 8; ++pr)
            if (at == (D == 128 ? kEnter128[pr] : kEnter64[pr]) + 2) {
                lrun0 += eb[pr][0];
                lrun1 += eb[pr][1];
                pw[pr] = pack_bf16x2(eb[pr][0], eb[pr][1]);
            }
#pragma unroll
        for (int pr = 0; pr < 8; ++pr)
            if (at == (D == 128 ? kEnter128[pr] : kEnter64[pr]) + 1) {
                eb[pr][0] = __builtin_amdgcn_exp2f(fa[pr][0]);
                eb[pr][1] = __builtin_amdgcn_exp2f(fa[pr][1]);
            }
#pragma unroll
        for (int pr = 0; pr < 8; ++pr)
            if (at == (D == 128 ? kEnter128[pr] : kEnter64[pr])) {
                fa[pr][0] = __builtin_fmaf(sc[2 * pr], a.scale_log2, -mrun);
                fa[pr][1] = __builtin_fmaf(sc[2 * pr + 1], a.scale_log2, -mrun);
            }
    };
    auto softmax_ahead = [&](const f32x16_t& sc) __attribute__((always_inline)) {      // what belongs into the step before a block's, at once
#pragma unroll
        for (int at = -NS; at < 0; ++at) softmax_slot(sc, at);
    };
    auto p_frag = [&](int st) __attribute__((always_inline)) {
        return __builtin_bit_cast(bf16x8_t, make_uint4(pw[4 * st], pw[4 * st + 1], pw[4 * st + 2], pw[4 * st + 3]));
    };
    // scores of keys that the row does not see (`vis`, shifted by 4 hi, has those it does): a quarter of a block's
    auto mask_piece = [&](f32x16_t& sn, int mi, uint32_t vis) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 4 * mi; i < 4 * mi + 4; ++i)
            if (!(vis >> ((i & 3) + 8 * (i >> 2)) & 1)) sn[i] = -__builtin_inff();
    };
    auto block_max = [&](const f32x16_t& sc) __attribute__((always_inline)) {      // of a row, times the scale
        float x = max3_tree(sc[0], sc[1], sc[2]), y = max3_tree(sc[3], sc[4], sc[5]);
        x = max3_tree(x, sc[6], sc[7]);
        y = max3_tree(y, sc[8], sc[9]);
        x = max3_tree(x, sc[10], sc[11]);
        y = max3_tree(y, sc[12], sc[13]);
        x = max3_tree(x, sc[14], sc[15]);
        const unsigned u = __float_as_uint(fmaxf(x, y) * a.scale_log2);
        const auto sw = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        return fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
    };
    bool exact = false;                // with a running maximum
    auto raise = [&](const f32x16_t& sc) __attribute__((always_inline)) {
        const float mloc = block_max(sc);
        if (__builtin_amdgcn_ballot_w64(mloc > mrun) != 0) {
            const float mnew = fmaxf(mrun, mloc), alpha = __builtin_amdgcn_exp2f(mrun - mnew);
            mrun = mnew;
            lrun0 *= alpha;
            lrun1 *= alpha;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) oacc[db][i] *= alpha;
        }
    };
    // Block u (scores sc, masked): weights, O += V^T P; scores of block u + 1 (keys at kblock) into sn.  kpre: its first reads, made
    // during the step before, refilled from kblock_after.  `dealt`: the first weights of block u + 1 in the slots too; else behind them, raised maximum
    // first where it runs.  hook(i): what else goes into slot i.
    bf16x8_t kpre[PF];
    auto block_step = [&](const f32x16_t& sc, f32x16_t& sn, const unsigned char* kblock, const unsigned char* vblock,
                          const unsigned char* kblock_after, uint32_t vis_next, auto hook, auto has_next, auto has_after, auto mask_next,
                          auto dealt) __attribute__((always_inline)) {
        constexpr bool kNext = decltype(has_next)::value, kAfter = decltype(has_after)::value, kDealt = decltype(dealt)::value;
        bf16x8_t kf[KS], vf[NP];
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (kNext) {
                if (i < PF) kf[i] = kpre[i];
                if (i + PF < KS) kf[i + PF] = k_frag(kblock, i + PF);
                const f32x16_t zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                sn = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[i], qf[i], i == 0 ? zero : sn, 0, 0, 0);
            }
            if (i + PFV >= KS) vf[i + PFV - KS] = v_frag(vblock, i + PFV - KS);
            softmax_slot(sc, i);
            hook(i);
        }
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            __builtin_amdgcn_sched_barrier(0);
            if (j + PFV < NP) vf[j + PFV] = v_frag(vblock, j + PFV);
            if constexpr (kAfter) {
                if (j + PF >= NP) kpre[j + PF - NP] = k_frag(kblock_after, j + PF - NP);
            }
            oacc[j % DB] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[j], p_frag(j / DB), oacc[j % DB], 0, 0, 0);
            softmax_slot(sc, KS + j);
            if constexpr (kNext && kDealt) softmax_slot(sn, j - NP);
            if constexpr (kNext && decltype(mask_next)::value) {
                if (j >= DB) {
#pragma unroll
                    for (int mi = (j - DB) * 4 / DB; mi < (j - DB + 1) * 4 / DB; ++mi) mask_piece(sn, mi, vis_next);
                }
            }
            hook(KS + j);
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (kNext && !kDealt) {
            if (exact) raise(sn);
            softmax_ahead(sn);
        }
    };
    const std::true_type yes{};
    const std::false_type no{};

    // ---- prologue: keys of KD and values of VD tiles asked for
    int64_t k_base, v_base[KD - VD];   // of tile t + KD; of tiles t + VD .., whose keys have been asked for
    int kslot, vslot;                  // slots: of tile t
    auto after = [](int slot, int step, int n) __attribute__((always_inline)) { return slot + step < n ? slot + step : slot + step - n; };
    auto tidy = [&](int t, int slot) __attribute__((always_inline)) {
        const uint64_t bits = counted(t);
        if (!open_tile(t, bits)) clean(slot, bits);
    };
    auto begin = [&]() __attribute__((always_inline)) {
        open_end = min(t1, s.ctx / KT);
        kslot = vslot = 0;
        fill(t0);
#pragma unroll
        for (int i = 0; i < KD; ++i) {
            const int64_t base = base_of(t0 + i);
#pragma unroll
            for (int n = 0; n < NI; ++n) copy_k(base, i, n);
            if (i < VD) {
#pragma unroll
                for (int n = 0; n < NI; ++n) copy_v(base, i, n);
            } else {
                v_base[i - VD] = base;
            }
        }
        // (the query rows' loads are waited for with the first tiles)
        wait_landed<(KD - 2) * NI + (VD - 1) * NI>();
        if (t0 >= open_end) tidy(t0, 0);
        __syncthreads();
    };
    // V(t + VD) and K(t + KD) into the slots that V(t - 1) and K(t - 1) left, in 2 NI pieces (values first, they are due first: 16 rows of 8191 keys, 64 nodes
    // of 8B heads 189 -> 185 us); in front of them the pages of the tiles to come
    auto look_ahead = [&](int t) __attribute__((always_inline)) {
        if (t + KD - tb > 63) fill(t);
    };
    auto request = [&](int t, int i) __attribute__((always_inline)) {
        if (i < NI) copy_v(v_base[0], after(vslot, VD, VD + 1), i);
        if (i == NI - 1) {
            k_base = base_of(t + KD);
#pragma unroll
            for (int n = 0; n + 1 < KD - VD; ++n) v_base[n] = v_base[n + 1];
            v_base[KD - VD - 1] = k_base;
        }
        if (i >= NI && i < 2 * NI) copy_k(k_base, after(kslot, KD, KD + 1), i - NI);
    };
    // the end of a tile: K(t + 2) and V(t + 1) have landed (what was asked for since the tile before may be on its way), values cleaned if need be
    auto turn = [&](int t, auto masks) __attribute__((always_inline)) {
        vslot = after(vslot, 1, VD + 1);
        kslot = after(kslot, 1, KD + 1);
        if constexpr (decltype(masks)::value) {
            wait_landed<(KD - 2) * NI + (VD - 1) * NI>();
            if (t + 1 >= open_end) tidy(t + 1, vslot);
            __syncthreads();
        } else {       // (a __syncthreads would wait for the next block's keys too, which nobody overwrites)
            asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" : : "n"((KD - 2) * NI + (VD - 1) * NI) : "memory");
        }
    };
    // behind the last tile: whether any wave left a value out (1), and whether any row left the safe range (2).  The word is the ring's first, which
    // nothing reads or writes any more
    auto report = [&](bool bad) __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // nothing may land in LDS behind this
        __syncthreads();
        int* flag = reinterpret_cast<int*>(ring);
        if (threadIdx.x == 0) *flag = 0;
        __syncthreads();
        if (odd || bad) atomicOr(flag, (odd ? 1 : 0) | (bad ? 2 : 0));
        __syncthreads();
        const int all = *flag;
        __syncthreads();
        return all;
    };
    if (!active) {       // a wave without rows stages its part of every tile
        for (int pass = 0; pass < 2; ++pass) {
            begin();
            for (int t = t0; t + 1 < t1; ++t) {
                look_ahead(t);
#pragma unroll
                for (int i = 0; i < 2 * NI; ++i) request(t, i);
                turn(t, yes);
            }
            if (!(report(false) & 2)) break;
        }
        if (KW == 2) __syncthreads();
        return;
    }
    auto mine = [&](uint64_t keys) __attribute__((always_inline)) -> uint64_t { return KW == 1 ? keys : keys >> (32 * kh) & 0xffffffffull; };

    f32x16_t s0, s1;
    auto nothing = [](int) {};
    auto tile_step = [&](int t, auto masks) __attribute__((always_inline)) {
        constexpr bool kMask = decltype(masks)::value;
        std::integral_constant<bool, !kMask> dealt;
        look_ahead(t);
        const unsigned char *kcur = kring + kslot * TB, *knext = kring + after(kslot, 1, KD + 1) * TB, *vcur = vring + vslot * TB;
        uint32_t vis1 = 0, vis2 = 0;
        if constexpr (kMask) {
            const uint64_t here = mine(visible(t, counted(t))), there = mine(visible(t + 1, counted(t + 1)));
            saw |= (here | there) != 0;
            vis1 = (uint32_t)(here >> 32) >> (4 * hi);
            vis2 = (uint32_t)there >> (4 * hi);
        }
        auto asks = [&](int i) __attribute__((always_inline)) { request(t, i); };
        static_assert(NS >= 2 * NI, "a request a slot");
        if constexpr (KW == 1) {
            block_step(s0, s1, kcur + 32 * RB, vcur, knext, vis1, asks, yes, yes, masks, dealt);
            block_step(s1, s0, knext, vcur + 32 * RB, knext + 32 * RB, vis2, nothing, yes, yes, masks, dealt);
        } else {
#pragma unroll
            for (int k = 0; k < PF; ++k) kpre[k] = k_frag(knext + kh * 32 * RB, k);
            block_step(s0, s1, knext + kh * 32 * RB, vcur + kh * 32 * RB, nullptr, vis2, asks, yes, no, masks, dealt);
            s0 = s1;
        }
        turn(t, masks);
    };
    int flags;
    while (true) {
        begin();
        mrun = kTreeNegBig;
        lrun0 = lrun1 = 0.f;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) oacc[db][i] = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) s0[i] = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k) s0 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k_frag(kring + kh * 32 * RB, k), qf[k], s0, 0, 0, 0);
        const uint64_t first = mine(visible(t0, counted(t0)));
        saw = first != 0;
#pragma unroll
        for (int mi = 0; mi < 4; ++mi) mask_piece(s0, mi, (uint32_t)first >> (4 * hi));
        if (exact) {
            raise(s0);
        } else {
            mrun = block_max(s0);
            if (!(fabsf(mrun) <= 3.4028235e38f)) mrun = 0.f;      // nothing seen yet
        }
        softmax_ahead(s0);
        if constexpr (KW == 1) {
#pragma unroll
            for (int k = 0; k < PF; ++k) kpre[k] = k_frag(kring + 32 * RB, k);
        }
        int t = t0;
        if (!exact)
            for (; t + 1 < open_end; ++t) tile_step(t, no);
        for (; t + 1 < t1; ++t) tile_step(t, yes);
        if constexpr (KW == 2) {
            block_step(s0, s1, nullptr, vring + vslot * TB + kh * 32 * RB, nullptr, 0, nothing, no, no, no, no);
        } else {   // the last tile: nothing follows its second block
            const uint32_t vis1 = (uint32_t)(visible(t, counted(t)) >> 32) >> (4 * hi);
            const unsigned char *kcur = kring + kslot * TB, *vcur = vring + vslot * TB;
            block_step(s0, s1, kcur + 32 * RB, vcur, nullptr, vis1, nothing, yes, no, yes, no);
            block_step(s1, s0, kcur, vcur + 32 * RB, nullptr, 0, nothing, no, no, no, no);
        }
        bool bad = false;
        if (!exact) {
            const float l = lrun0 + lrun1 + __shfl_xor(lrun0 + lrun1, 32, 64);
            bad = saw && !(l >= 0x1p-20f && l <= 0x1p64f);
            float none = 0.f;      // zero unless a sum is not finite
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) none = fmaf(oacc[db][i], 0.f, none);
            bad |= none != 0.f;
        }
        flags = report(bad);
        if (exact || !(flags & 2)) break;
        exact = true;
    }
    if (!saw) mrun = kTreeNegBig;
    float den = lrun0 + lrun1 + __shfl_xor(lrun0 + lrun1, 32, 64);
    if constexpr (KW == 2) {       // the states of a row's two waves: lane by lane through the ring
        constexpr int EACH = DB * 16 + 4;
        float* at = reinterpret_cast<float*>(ring) + (rg * 64 + lane) * EACH;
        if (kh == 1) {
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *reinterpret_cast<f32x4_t*>(at + db * 16 + i) = (f32x4_t){oacc[db][i], oacc[db][i + 1], oacc[db][i + 2], oacc[db][i + 3]};
            at[DB * 16] = mrun;
            at[DB * 16 + 1] = den;
        }
        __syncthreads();
        if (kh == 1) return;
        const float m1 = at[DB * 16], top = fmaxf(mrun, m1), f0 = __builtin_amdgcn_exp2f(mrun - top), f1 = __builtin_amdgcn_exp2f(m1 - top);
        den = fmaf(at[DB * 16 + 1], f1, den * f0);
        mrun = top;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const f32x4_t o = *reinterpret_cast<const f32x4_t*>(at + db * 16 + i);
#pragma unroll
                for (int j = 0; j < 4; ++j) oacc[db][i + j] = fmaf(o[j], f1, oacc[db][i + j] * f0);
            }
    }
    if (!stored) return;
    // oacc[db][i] = O^T[32 db + (i & 3) + 8 (i >> 2) + 4 hi][row]
    if (flags & 1)
        odd_values<false, D>(a, s, b, kvh, node, t0 * KT, 1 << 30, 1 << 30, min(t1 * KT, s.total), KT, [&](const uint16_t* v) {
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const f32x4_t x = TreeT<false>::ld4(v + 32 * db + 8 * k + 4 * hi);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (is_odd(x[j])) oacc[db][4 * k + j] += x[j];
                }
        });
    const bool whole = splits == 1;
    const int64_t tok = s.start + node;
    const float inv = den != 0.f ? 1.0f / den : 0.f;
    const int64_t at = ((int64_t)split * a.tokens + tok) * a.hq + head;
    uint16_t* op = (uint16_t*)a.out + tok * a.ldo + (int64_t)head * D + 4 * hi;
    float* pp = a.part + at * D + 4 * hi;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const f32x4_t o = {oacc[db][4 * k], oacc[db][4 * k + 1], oacc[db][4 * k + 2], oacc[db][4 * k + 3]};
            if (whole) TreeT<false>::st4(op + 32 * db + 8 * k, o * inv);
            else *reinterpret_cast<f32x4_t*>(pp + 32 * db + 8 * k) = o;
        }
    if (!whole && hi == 0) {
        a.state[2 * at] = mrun;
        a.state[2 * at + 1] = den;
    }
}

// Splits added in order; rows that one split holds are written already.  A (node, head) is 2^shift groups of D / 4 lanes, each of which adds every
// 2^shift-th split with all its requests out at once (64 splits in one group: 32 dependent trips, 17 us where this takes 4).
template <bool F32, int D>
__global__ __launch_bounds__(256) void tree_attn_merge_kernel(TreeArgs a) {
    typedef TreeT<F32> X;
    constexpr int LPR = D / 4, GROUPS = 256 / LPR, MOST = 4;
    __shared__ float topL[GROUPS], denL[GROUPS];
    __shared__ f32x4_t oL[256];
    const int b = blockIdx.y, group = threadIdx.x / LPR, c = threadIdx.x % LPR * 4;
    const TreeWork work = step_work(a);
    const TreeSpan s = tree_span(a, b);
    const int filled = row_splits(a, s.total, work);
    if (filled <= 1) return;
    int shift = 0;
    while ((MOST << shift) < filled && (1 << shift) < GROUPS) ++shift;
    const int part = group & ((1 << shift) - 1), each = GROUPS >> shift, items = s.n * a.hq;
    const int64_t step = (int64_t)a.tokens * a.hq;
    for (int base = blockIdx.x * each; base < items; base += gridDim.x * each) {      // (the same trips for the whole workgroup)
        const int item = base + (group >> shift), node = min(item / a.hq, s.n - 1), head = item % a.hq;
        const int64_t t = s.start + node, at = t * a.hq + head;
        float top = kTreeNegBig, den = 0.f;
        f32x4_t o = {0.f, 0.f, 0.f, 0.f};
        for (int first = part; first < filled; first += MOST << shift) {
            float m[MOST], l[MOST];
            f32x4_t x[MOST];
#pragma unroll
            for (int i = 0; i < MOST; ++i) {
                m[i] = -__builtin_inff();
                if (first + (i << shift) >= filled) continue;
                const int64_t from = at + (first + (i << shift)) * step;
                m[i] = a.state[2 * from];
                l[i] = a.state[2 * from + 1];
                x[i] = *reinterpret_cast<const f32x4_t*>(a.part + from * D + c);
            }
            float up = top;
#pragma unroll
            for (int i = 0; i < MOST; ++i) up = fmaxf(up, m[i]);
            const float f0 = __builtin_amdgcn_exp2f(top - up);
            den *= f0;
            o *= f0;
            top = up;
#pragma unroll
            for (int i = 0; i < MOST; ++i) {
                if (first + (i << shift) >= filled) break;
                const float f = __builtin_amdgcn_exp2f(m[i] - top);
                den = fmaf(l[i], f, den);
                o += x[i] * f;
            }
        }
        if (shift > 0) {
            if (c == 0) {
                topL[group] = top;
                denL[group] = den;
            }
            oL[threadIdx.x] = o;
            __syncthreads();
            float up = top;
            for (int i = 1; i < 1 << shift; ++i) up = fmaxf(up, topL[min(group + i, GROUPS - 1)]);
            const float f0 = __builtin_amdgcn_exp2f(top - up);
            den *= f0;
            o *= f0;
            for (int i = 1; i < 1 << shift; ++i) {
                const int from = min(group + i, GROUPS - 1);
                const float f = __builtin_amdgcn_exp2f(topL[from] - up);
                den = fmaf(denL[from], f, den);
                o += oL[from * LPR + threadIdx.x % LPR] * f;
            }
            __syncthreads();      // (the next items' states go to the same places)
        }
        if (part != 0 || item >= items) continue;
        const float inv = den != 0.f ? 1.0f / den : 0.f;
        X::st4((typename X::T*)a.out + t * a.ldo + (int64_t)head * D + c, o * inv);
    }
}

// Which kernel a launch takes, with rows, workgroups and keys of its workgroups.  max_keys is what the table has room for: nothing is read back, and a table of
// more columns than the rows want costs a short row up to twice its time (the shim's caller can pass fewer columns).
// Where few workgroups have short rows, latency counts: a workgroup of 16 stacked rows is the quickest through its keys, and as many of them as the chip
// has units ask for the same keys again out of L2.  Past `reach` (workgroups times keys) that traffic is what they take, and a workgroup takes more rows:
// 32, then 64 (heads of 64), then the wide form.  In us, 16 rows a workgroup, 32, wide, each with the splits that it gets:
//   32 heads of 64 on 4     1 row of 600, 64 nodes 8.2, 10.7, 16.4; 4 rows of 1200, 32 nodes 11.1, 14.2, 20.3; 64 nodes 17.1, 14.7, 20.7; of 5000, 16 nodes
//                           21.5, 20.0, 19.9; 64 nodes 54, 44, 32; 32 rows of 1200, 8 nodes 17.1, 15.5, 20.1
//   32 heads of 128 on 8    1 row of 600, 64 nodes 11.3, 15.3, 19.2; 1200 15.0, 18.4, 21.4; 2500 20.9, 21.9, 21.8; 2 rows of 1900 20.5, 24.2, 23.0; 4 rows of
//                           1200, 32 nodes 15.7, 20.6, 24.7; 64 nodes 29, 21, 27; 2500 57, 38, 30; 16 rows of 1200, 16 nodes 31.7, 21.9, 26.5
// Where every other form has passed its reach: 64 rows a workgroup for heads of 64 (32 rows of 4096, 8 nodes 34.5, wide 36.9), else wide; 32 rows of heads of
// 128 in the narrow form (107, wide 120).  fp32, whose blocks are bound by their matrix instructions, 16 or 32 rows by the same rule (4 rows of 2500, 16 heads
// of 64 on 4, 16 nodes 18.4, 21.7; 64 nodes of heads of 128 75, 66).
struct TreeForm {
    int row_tiles, row_part, row_blocks, round_keys, wide, waves, deep, whole, per_unit, slots, least;
};
static TreeForm tree_form(int rows, int max_nodes, int hkv, int g, int d, int f32, int64_t max_keys) {
    const int64_t stacked = (int64_t)max_nodes * g, heads = (int64_t)rows * hkv;
    auto fits = [&](int tiles, int most, int64_t reach) {
        const int64_t wgs = heads * ((stacked + 16 * tiles - 1) / (16 * tiles));
        return wgs <= most && wgs * max_keys <= reach;
    };
    TreeForm f;
    f.wide = 0;
    const bool few = max_keys <= (d == 64 ? 1536 : 2304);
    if (f32) f.row_tiles = stacked <= 16 || fits(1, num_cus(), 400000) ? 1 : 2;
    else if (stacked <= 16 || fits(1, num_cus(), d == 64 ? few ? 400000 : 200000 : few ? 600000 : 250000)) f.row_tiles = 1;
    else if (stacked <= 32 || fits(2, num_cus(), max_keys <= 1536 ? 400000 : 250000)) f.row_tiles = 2;
    else f.row_tiles = 4, f.wide = d == 128 || stacked > 64;
    f.row_part = f.wide ? (stacked <= 64 ? 64 : 128) : 16 * f.row_tiles;
    f.row_blocks = (int)((stacked + f.row_part - 1) / f.row_part);
    // (16 rows of heads of 128: what a compute unit has on its way is what it gets through; eight waves have twice as much.  8 heads of 128 on 1, 16 nodes, four
    // and eight: 45 keys 6.4, 6.7; 300 8.9, 8.3; 2500 in one piece 26.5, 21.5; one row of 4096 of 32 on 8 17.2, 15.9.  Heads of 64 gain nothing)
    // So have 32 rows of heads of 64 that are not cut (below): 4 rows of 1200, 64 nodes 15.0, 13.8; cut they are slower for it, 16 nodes of 2500 15.5, 16.8.
    const bool half = 2 * heads * f.row_blocks >= num_cus();      // a workgroup for every other unit
    f.waves = !f32 && !f.wide && ((d == 128 && f.row_tiles == 1 && max_keys > 256) || (d == 64 && f.row_tiles == 2 && half && max_keys <= 6144)) ? 8 : 4;
    f.whole = f.waves == 8 && half && max_keys <= (d == 64 ? 6144 : 2304);
    // 64 rows of heads of 128 go through a tile in less time than memory answers in: where there is one workgroup a unit or nearly, keys three tiles ahead
    // instead of two (112 KB of LDS) and rows whole: 32 rows of 4000, 16 nodes of 8B heads 119 -> 103 us, uneven ones 71 -> 65; 24 rows 97 -> 85, uneven
    // 49 -> 51; 18 uneven ones would be 39 -> 46.  (With 128 rows the compiler then moves accumulators between its two files of registers, 17 % slower.)
    f.deep = f.wide && f.row_part == 64 && 4 * heads * f.row_blocks >= 3 * num_cus() && heads * f.row_blocks <= num_cus() && max_keys <= 6144;
    f.whole |= f.deep;
    f.round_keys = f.wide || f32 ? 64 : 32 * f.waves;
    // Work for one workgroup a unit, or for two where there are two without any cut (wide, us with one and two: 32 uneven rows of 256 to 8191, 64
    // nodes of 8B heads 203, 199; 16 nodes 151, 159; one row of 8191, 64 nodes 29.4, 33.5; 16 rows of 4000, 32 nodes 63.7, 70.4).  fp32 by workgroups times
    // keys, us with one and two: under 100000 one is quicker (16 nodes of 16 heads of 64 on 4, one row of 3000 12.9, 14.6, two 15.4, 15.9; of 8 heads of 128 14.1, 16.0
    // and 18.8, 20.8); from there to 200000 either (three rows 21.6, 18.4, four 19.5, 20; four of 8 heads of 128 25.2, 26.6); above it two by up to a quarter, one by 7 % in
    // some (24 rows of 240 to 4000, 16 nodes, 8 heads of 64 52, 46, of 128 133, 100; 4 of 4000, 24 nodes, 16 heads of 128 on 8 77, 65; 8 of 3000, 16 nodes, 8 heads of 64
    // 23.5, 23.9, of 128 39, 41; 16 of 480 to 8000, 4 nodes, 32 heads of 64 on 8 61, 69)
    const bool two = f.wide ? heads * f.row_blocks >= 2 * num_cus()
                            : f32 && (d == 64 || f.row_tiles == 1) && heads * f.row_blocks * max_keys >= 200000;
    f.per_unit = two ? 2 : 1;
    f.slots = num_cus() * f.per_unit;
    f.least = f.wide ? 6 : 1;
    return f;
}

}  // namespace mv

extern "C" {

size_t mv_tree_attn_workspace_bytes(int tokens, int hq, int d, int num_splits) {
    if (tokens <= 0 || hq <= 0 || d <= 0 || num_splits <= 1) return 0;
    return (size_t)num_splits * tokens * hq * (d + 2) * sizeof(float);
}

int mv_tree_attn_pick_splits(int rows, int max_nodes, int hq, int hkv, int d, int max_keys, int f32) {
    using namespace mv;
    if (rows <= 0 || max_nodes <= 0 || hq <= 0 || hkv <= 0 || hq % hkv || max_keys <= 0) return 1;
    const TreeForm f = tree_form(rows, max_nodes, hkv, hq / hkv, d, f32, max_keys);
    // the launch that joins the splits costs some 3 us, a round of a workgroup 0.5 (heads of 64) to 1.2 (of 128): short rows are not cut (heads of 64,
    // one row of 1200, 64 nodes whole 10.7, cut 12.5, of 2500 17.3, 16.0; heads of 128 of 600 14.4, 15.8, of 1200, 16 nodes 18.3,
    // 14.4; fp32, 8 heads of 64 of 300 8.3, 10.1, of 600 12.1, 10.6)
    if (max_keys <= (f32 ? 512 : d == 64 ? 1536 : 1024)) return 1;
    // (nor rows that workgroups of eight waves are through with soon, of which there is one for every other unit: 4 rows of 1200, 16 nodes of 8B heads 14.6,
    // 17.3; 2 rows of 1900, 64 nodes 20.5, 27.0; 32 rows of 5000, 4 nodes, 32 heads of 64 on 4 32, 36)
    if (f.whole) return 1;
    // (as many as the kernels may want: they cut a row in fewer where its keys or the step's rows do not ask for them)
    const int64_t units = (int64_t)rows * hkv * f.row_blocks, most = ((int64_t)max_keys + f.round_keys * f.least - 1) / (f.round_keys * f.least);
    // Rows enough for every slot are cut for the sake of long ones among short ones, where the longest that the table has room for would last: what is
    // not cut is 7 to 15 % quicker where the rows are alike (64 rows of 2048, 8 nodes 64, 69; 512 rows, 2 nodes 432, 475).  fp32: one workgroup a unit is
    // enough (4 rows of 900, 64 nodes, 16 heads of 128 on 4 whole 31, cut 38).
    int64_t splits = units < (f32 ? num_cus() : f.slots) ? (f.slots + units - 1) / units * (rows > 1 ? 2 : 1)
                     : max_keys >= 4096 && max_keys >= 1024 * units / f.slots ? 4 : 1;
    if (rows == 1 && units >= f.slots) splits = 1;
    if (splits > most) splits = most;
    if (splits > 1 && (int64_t)rows * hkv * splits > 8 * 65535) splits = 1;      // (the grid's third dimension)
    return (int)(splits < 1 ? 1 : splits > kTreeMaxSplits ? kTreeMaxSplits : splits);
}

int mv_tree_attn(const void* q, int64_t ldq, const void* k_cache, const void* v_cache, const int32_t* ctx_lens, const int32_t* row_start,
                 const int32_t* block_table, int64_t bt_stride, int bt_cols, const uint64_t* mask, int words, void* out, int64_t ldo,
                 void* workspace, size_t workspace_bytes, int rows, int tokens, int max_nodes, int hq, int hkv, int d, int page,
                 int num_pages, float scale, int num_splits, int f32, mv_stream_t stream) {
    using namespace mv;
    if (rows < 0 || tokens < 0 || max_nodes < 0 || hq <= 0 || hkv <= 0 || hq % hkv || page <= 0 || num_pages <= 0 || bt_cols <= 0 ||
        bt_stride < bt_cols || num_splits < 1 || !(scale > 0.f) || scale > 3.0e38f)
        return MV_ERR_INVALID_ARG;
    if ((d != 64 && d != 128) || hq / hkv > 8 || (page & (page - 1)) || page < kTreeBlock || max_nodes > kTreeMaxNodes || num_splits > kTreeMaxSplits)
        return MV_ERR_UNSUPPORTED;
    if (((int64_t)bt_cols << __builtin_ctz((unsigned)page)) > (1 << 30)) return MV_ERR_UNSUPPORTED;      // (an index of a key, and what is added to it, has 32 bits)
    if (rows == 0 || tokens == 0 || max_nodes == 0) return MV_OK;
    if (!q || !k_cache || !v_cache || !ctx_lens || !row_start || !block_table || !out) return MV_ERR_INVALID_ARG;
    if (mask && (words < 1 || words > kTreeMaxWords || words * 64 < max_nodes)) return MV_ERR_INVALID_ARG;
    const int vec = f32 ? 4 : 8;
    if (ldq < (int64_t)hq * d || ldo < (int64_t)hq * d || ldq % vec || ldo % vec || !aligned16(q) || !aligned16(out) ||
        !aligned16(k_cache) || !aligned16(v_cache))
        return MV_ERR_INVALID_ARG;
    if (num_splits > 1 && (!workspace || !aligned16(workspace) || workspace_bytes < mv_tree_attn_workspace_bytes(tokens, hq, d, num_splits)))
        return MV_ERR_WORKSPACE;
    const int64_t bytes = f32 ? 4 : 2;
    if (rows_meet(q, ldq * bytes, hq * d * bytes, out, ldo * bytes, hq * d * bytes, tokens)) return MV_ERR_INVALID_ARG;
    // neither the output nor the partial sums may lie over what other workgroups still read (the table as from its first to its last column)
    const int64_t row = hq * d * bytes, pool = (int64_t)num_pages * page * hkv * d * bytes;
    const MemSpan part[] = {{num_splits > 1 ? workspace : nullptr, (int64_t)mv_tree_attn_workspace_bytes(tokens, hq, d, num_splits)}};
    const MemSpan ins[] = {{k_cache, pool}, {v_cache, pool}, {ctx_lens, (int64_t)rows * 4}, {row_start, (int64_t)rows * 4 + 4},
                           {mask, (int64_t)tokens * words * 8}, {block_table, ((rows - 1) * bt_stride + bt_cols) * 4}};
    if (outputs_meet(part, ins) || rows_meet_span(q, ldq * bytes, row, tokens, part[0].p, part[0].n) ||
        rows_meet_span(out, ldo * bytes, row, tokens, part[0].p, part[0].n))
        return MV_ERR_INVALID_ARG;
    for (const MemSpan& s : ins)
        if (rows_meet_span(out, ldo * bytes, row, tokens, s.p, s.n)) return MV_ERR_INVALID_ARG;
    TreeArgs a;
    a.q = q;
    a.k_cache = k_cache;
    a.v_cache = v_cache;
    a.ldq = ldq;
    a.ctx = ctx_lens;
    a.row_start = row_start;
    a.block_table = block_table;
    a.bt_stride = bt_stride;
    a.mask = mask;
    a.words = words;
    a.out = out;
    a.ldo = ldo;
    a.part = (float*)workspace;
    a.state = num_splits > 1 ? (float*)workspace + (size_t)num_splits * tokens * hq * d : nullptr;
    a.bt_cols = bt_cols;
    a.rows = rows;
    a.tokens = tokens;
    a.max_nodes = max_nodes;
    a.hq = hq;
    a.hkv = hkv;
    a.g = hq / hkv;
    a.page = page;
    a.page_shift = __builtin_ctz((unsigned)page);
    a.num_pages = num_pages;
    a.nsplit = num_splits;
    const TreeForm f = tree_form(rows, max_nodes, hkv, a.g, d, f32, (int64_t)bt_cols << a.page_shift);
    a.row_blocks = f.row_blocks;
    a.round_keys = f.round_keys;
    a.row_part = f.row_part;
    a.slots = f.slots;
    a.least = f.least;
    a.per_unit = f.per_unit;
    a.scale_log2 = scale * 1.4426950408889634f;
    const int64_t places = (int64_t)rows * hkv * num_splits, together = places >= 8 ? 8 : 1, high = (places + together - 1) / together;
    if (high > 65535 || rows > 65535) return MV_ERR_UNSUPPORTED;
    hipStream_t s = (hipStream_t)stream;
    const dim3 g1((unsigned)together, (unsigned)a.row_blocks, (unsigned)high);
#define MV_TREE(K_) hipLaunchKernelGGL((K_), g1, dim3((unsigned)f.waves * 64), 0, s, a)
    if (f32 && d == 64 && f.row_tiles == 1) MV_TREE((tree_attn_f32_kernel<64, 1>));
    else if (f32 && d == 64) MV_TREE((tree_attn_f32_kernel<64, 2>));
    else if (f32 && f.row_tiles == 1) MV_TREE((tree_attn_f32_kernel<128, 1>));
    else if (f32) MV_TREE((tree_attn_f32_kernel<128, 2>));
    else if (f.wide && d == 64) MV_TREE((tree_attn_wide_kernel<64, 1, 4>));      // (64 rows of such heads: the narrow form)
    else if (f.wide && f.row_part == 64 && f.deep) MV_TREE((tree_attn_wide_kernel<128, 2, 3>));
    else if (f.wide && f.row_part == 64) MV_TREE((tree_attn_wide_kernel<128, 2, 2>));
    else if (f.wide) MV_TREE((tree_attn_wide_kernel<128, 1, 2>));
    else if (d == 64 && f.row_tiles == 1) MV_TREE((tree_attn_narrow_kernel<64, 1, 4>));
    else if (d == 64 && f.row_tiles == 2 && f.waves == 8) MV_TREE((tree_attn_narrow_kernel<64, 2, 8>));
    else if (d == 64 && f.row_tiles == 2) MV_TREE((tree_attn_narrow_kernel<64, 2, 4>));
    else if (d == 64) MV_TREE((tree_attn_narrow_kernel<64, 4, 4>));
    else if (f.row_tiles == 1 && f.waves == 8) MV_TREE((tree_attn_narrow_kernel<128, 1, 8>));
    else if (f.row_tiles == 1) MV_TREE((tree_attn_narrow_kernel<128, 1, 4>));
    else MV_TREE((tree_attn_narrow_kernel<128, 2, 4>));
#undef MV_TREE
    if (num_splits > 1) {
        const int groups = 1024 / d;
        int shift = 0;
        while ((4 << shift) < num_splits && (1 << shift) < groups) ++shift;      // (as the kernel at most)
        // (rows that are not cut leave at once, but a workgroup that leaves has asked for lengths too: no more of them than the chip holds: 8 rows of 8191
        // keys, 48 nodes, 8 heads of 128 on 1 33.8 us, with twice as many 35.5)
        const int64_t most = ((int64_t)max_nodes * hq + (groups >> shift) - 1) / (groups >> shift), fair = (8 * num_cus() + rows - 1) / rows;
        const dim3 g2((unsigned)(most < fair ? most : fair), (unsigned)rows);
        if (f32 && d == 64) hipLaunchKernelGGL((tree_attn_merge_kernel<true, 64>), g2, dim3(256), 0, s, a);
        else if (f32) hipLaunchKernelGGL((tree_attn_merge_kernel<true, 128>), g2, dim3(256), 0, s, a);
        else if (d == 64) hipLaunchKernelGGL((tree_attn_merge_kernel<false, 64>), g2, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((tree_attn_merge_kernel<false, 128>), g2, dim3(256), 0, s, a);
    }
    return check_launch();
}

}  // extern "C"
