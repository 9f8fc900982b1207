// What stands around the attention of a step that verifies drafted tokens (tree_attn.hip): its plan, the store of its keys and
// values, and the acceptance.  Row b brings nodes row_start[b] .. row_start[b + 1] - 1 behind ctx[b] cached tokens; node i lies at
// index ctx[b] + i of its sequence, whatever its depth; a parent is an earlier node of the row (anything else: none).
//
//   tree_plan              pages for the nodes from a free list, slots, positions (ctx + depth), ancestor masks
//   qkv_norm_rotary_slots  RMS norm of every head of q and k, rotation by position, keys and values to their slots
//   tree_accept            the walk from node 0 along the target's picks; the accepted nodes' keys and values moved to
//                          indices ctx .. of their sequence in every layer
#include "common.h"

namespace mv {

constexpr int kTreeNodes = 256;                // nodes of a row with a tree or a mask
constexpr int kTreeWords = kTreeNodes / 64;

struct TreeRow {
    int start, n, end;       // end: of all its nodes, n: of those within the bound
};
// nodes of row b, kept inside the step's tokens and the caller's bound whatever row_start holds
__device__ __forceinline__ TreeRow tree_row(const int32_t* row_start, int b, int tokens, int max_nodes) {
    const int s = min(max(row_start[b], 0), tokens), e = min(max(row_start[b + 1], s), tokens);
    return {s, min(e - s, max_nodes), e};
}

// ------------------------------------------------------------------ plan

struct PlanArgs {
    const int32_t *ctx, *row_start, *parents, *free_pages;
    int32_t* block_table;
    int64_t bt_stride;
    int bt_cols, n_free, rows, tokens, max_nodes, page, num_pages, words;
    int32_t *slots, *positions, *row_of, *taken;
    uint64_t* mask;
};

struct PageNeed {
    int64_t held, total;     // pages of the cached tokens, and with the nodes
    bool wide;               // the table has no column for them
    __device__ int64_t need() const { return wide ? 0 : total - held; }
};
__device__ __forceinline__ PageNeed page_need(const PlanArgs& a, int b) {
    const int64_t c = max(a.ctx[b], 0);
    const int n = tree_row(a.row_start, b, a.tokens, a.max_nodes).n;
    PageNeed p;
    p.held = (c + a.page - 1) / a.page;
    p.total = n > 0 ? (c + n + a.page - 1) / a.page : p.held;
    p.wide = p.total > a.bt_cols;
    return p;
}

// One workgroup per row (and, for rows without tree or mask, per chunk of blockDim.x nodes).  Every workgroup sums the needs of the
// rows before its own itself: two dependent trips to the caches for any number of rows, where a scan in a launch of its own is a
// launch.  Ancestors by doubling: a node's bits and its ancestor 2^k steps up; after k + 1 rounds it holds 2^(k + 1) of them, and the
// rounds end when every pointer has left the tree.
// The store behind the plan goes by slots alone, so tokens that no row has (in front of the first, behind the last, past a row's bound) may not keep
// the place that an earlier step's node had: their slot becomes -1, unless it is negative already.
__global__ __launch_bounds__(256) void tree_plan_kernel(PlanArgs a) {
    __shared__ int64_t red[4];
    __shared__ uint64_t bitsL[kTreeWords][kTreeNodes];
    __shared__ int upL[kTreeNodes];
    const int b = blockIdx.x, tid = threadIdx.x, nt = blockDim.x;
    const TreeRow row = tree_row(a.row_start, b, a.tokens, a.max_nodes);
    const int64_t ctx = max(a.ctx[b], 0);
    const PageNeed own = page_need(a, b);
    const int first = max(a.row_start[0], 0), last = max(a.row_start[a.rows], 0);

    int64_t before = 0;
    for (int i = tid; i < b; i += nt) before += page_need(a, i).need();
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) before += __shfl_xor(before, o, 64);
    if (nt > 64) {
        if ((tid & 63) == 0) red[tid >> 6] = before;
        __syncthreads();
        before = 0;
        for (int i = 0; i < nt / 64; ++i) before += red[i];
    }
    const bool refused = own.wide || (own.need() > 0 && before + own.need() > a.n_free);
    int32_t* table = a.block_table + (int64_t)b * a.bt_stride;
    if (blockIdx.y == 0) {
        if (tid == 0) a.taken[b] = refused ? -1 : (int)own.need();
        // (a refused row's columns may name pages that were given back since, and that another row takes here)
        const int64_t end = min(own.total, (int64_t)a.bt_cols);
        for (int64_t j = own.held + tid; j < end; j += nt) table[j] = refused ? -1 : a.free_pages[before + j - own.held];
    }

    const int i = blockIdx.y * nt + tid;
    int depth = i;
    if (a.mask || a.parents) {       // one chunk holds the row
        int up = -1;
        uint64_t bits[kTreeWords];
        if (i < row.n) {
            const int p = a.parents ? a.parents[row.start + i] : i - 1;
            up = p >= 0 && p < i ? p : -1;
        }
#pragma unroll
        for (int w = 0; w < kTreeWords; ++w) bits[w] = (i >> 6) == w ? 1ull << (i & 63) : 0;
        if (a.parents) {
            while (true) {
                upL[tid] = up;
#pragma unroll
                for (int w = 0; w < kTreeWords; ++w)
                    if (w < a.words) bitsL[w][tid] = bits[w];
                if (!__syncthreads_or(up >= 0)) break;
                if (up >= 0) {
#pragma unroll
                    for (int w = 0; w < kTreeWords; ++w)
                        if (w < a.words) bits[w] |= bitsL[w][up];
                    up = upL[up];
                }
                __syncthreads();
            }
            depth = -1;
#pragma unroll
            for (int w = 0; w < kTreeWords; ++w) depth += __popcll(bits[w]);
        } else {
#pragma unroll
            for (int w = 0; w < kTreeWords; ++w) {
                const int k = i + 1 - 64 * w;      // a chain: everything up to the node
                bits[w] = k >= 64 ? ~0ull : k > 0 ? (1ull << k) - 1 : 0;
            }
        }
        if (i < row.n && a.mask) {
#pragma unroll
            for (int w = 0; w < kTreeWords; ++w)
                if (w < a.words) a.mask[(int64_t)(row.start + i) * a.words + w] = bits[w];
        }
    }
    if (first > 0 || row.start + row.n < row.end || last < a.tokens) {
        const auto none = [&](int64_t t, int64_t end, int64_t step) {
            for (; t < end; t += step)
                if (a.slots[t] >= 0) a.slots[t] = -1;
        };
        const int wide = gridDim.y * nt;
        const int64_t nth = (int64_t)b * wide + i, all = (int64_t)gridDim.x * wide;
        none(nth, min(first, a.tokens), all);
        none((int64_t)row.start + row.n + i, row.end, wide);
        none(last + nth, a.tokens, all);
    }
    if (i >= row.n) return;
    const int64_t at = ctx + i, col = at / a.page;
    int slot = -1;
    if (!refused) {
        const int pg = col < own.held ? table[col] : a.free_pages[before + col - own.held];
        if (pg >= 0 && pg < a.num_pages) slot = pg * a.page + (int)(at % a.page);
    }
    const int64_t t = row.start + i;
    a.slots[t] = slot;
    a.positions[t] = (int)(ctx + depth);
    a.row_of[t] = b;
}

// ------------------------------------------------------------------ norm, rotation, store

template <bool F32> struct RowT;
template <> struct RowT<true> {
    typedef float T;
    static __device__ __forceinline__ float ld(const float* p) { return *p; }
    static __device__ __forceinline__ void st(float* p, float v) { *p = v; }
};
template <> struct RowT<false> {
    typedef uint16_t T;
    static __device__ __forceinline__ float ld(const uint16_t* p) { return bf16_bits_to_f32(*p); }
    static __device__ __forceinline__ void st(uint16_t* p, float v) { *p = (uint16_t)f32_to_bf16_bits(v); }
};

struct SlotStoreArgs {
    const void* qkv;
    int64_t ld;
    const float *q_norm, *k_norm;
    float eps;
    const double* inv_freq;
    int rot, adjacent;
    const int32_t *positions, *slots;
    void* q_out;
    int64_t ldq;
    void *k_cache, *v_cache;
    int tokens, hq, hkv, d;
    int64_t slots_n;      // slots of the cache
};

// sin and cos of pos * inv_freq.  The angle is formed and brought to [-1/2, 1/2] quarter turns in fp64 (a far position's angle has no
// bits left for that in fp32), the series of the remaining |x| <= pi / 4 run in fp32: sin to x^11, cos to x^10, the next terms below 2^-30.
__device__ __forceinline__ void sincos_turn(int pos, double inv_freq, float& sn, float& cs) {
    const double quarters = (double)pos * inv_freq * 0.63661977236758134308;
    const double whole = rint(quarters);
    const float x = (float)((quarters - whole) * 1.57079632679489661923), x2 = x * x;
    float s = fmaf(x2, -2.5052108e-8f, 2.7557319e-6f);
    s = fmaf(x2, s, -1.9841270e-4f);
    s = fmaf(x2, s, 8.3333333e-3f);
    s = fmaf(x2, s, -1.6666667e-1f);
    s = fmaf(x * x2, s, x);
    float c = fmaf(x2, -2.7557319e-7f, 2.4801587e-5f);
    c = fmaf(x2, c, -1.3888889e-3f);
    c = fmaf(x2, c, 4.1666667e-2f);
    c = fmaf(x2, c, -0.5f);
    c = fmaf(x2, c, 1.0f);
    const int quad = (int)((int64_t)whole & 3);
    const float a = quad & 1 ? c : s, b = quad & 1 ? s : c;
    sn = quad & 2 ? -a : a;
    cs = quad == 1 || quad == 2 ? -b : b;
}

// Any head size, alignment and rotated part: a wave per (token, head), its values read twice.
template <bool SF32, bool DF32>
__global__ __launch_bounds__(256) void slot_store_any_kernel(SlotStoreArgs a) {
    typedef RowT<SF32> S;
    typedef RowT<DF32> O;
    const int units = a.hq + 2 * a.hkv, lane = threadIdx.x & 63, d = a.d, half = a.rot / 2;
    const int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (wave >= (int64_t)a.tokens * units) return;
    const int64_t t = wave / units;
    const int u = (int)(wave % units);
    const typename S::T* x = (const typename S::T*)a.qkv + t * a.ld + (int64_t)u * d;
    const int64_t slot = a.slots[t];
    typename O::T* dst;
    if (u < a.hq) {
        dst = (typename O::T*)a.q_out + t * a.ldq + (int64_t)u * d;
    } else {
        if (slot < 0 || slot >= a.slots_n) return;
        const bool is_v = u >= a.hq + a.hkv;
        dst = (typename O::T*)(is_v ? a.v_cache : a.k_cache) + (slot * a.hkv + (u - a.hq - (is_v ? a.hkv : 0))) * d;
    }
    if (u >= a.hq + a.hkv) {
        for (int c = lane; c < d; c += 64) O::st(dst + c, S::ld(x + c));
        return;
    }
    const float* w = u < a.hq ? a.q_norm : a.k_norm;
    float inv = 1.f;
    if (w) {
        float ss = 0.f;
        for (int c = lane; c < d; c += 64) {
            const float v = S::ld(x + c);
            ss = fmaf(v, v, ss);
        }
        inv = 1.0f / sqrtf(wave_sum(ss) / (float)d + a.eps);
    }
    for (int j = lane; j < d - half; j += 64) {       // a head's pairs, then its other values
        if (j < half) {
            const int e0 = a.adjacent ? 2 * j : j, e1 = a.adjacent ? 2 * j + 1 : j + half;
            float sn, cs;
            sincos_turn(a.positions[t], a.inv_freq[j], sn, cs);
            float x0 = S::ld(x + e0) * inv, x1 = S::ld(x + e1) * inv;
            if (w) x0 *= w[e0], x1 *= w[e1];
            O::st(dst + e0, x0 * cs - x1 * sn);
            O::st(dst + e1, x1 * cs + x0 * sn);
        } else {
            const int e = half + j;
            const float v = S::ld(x + e) * inv;
            O::st(dst + e, w ? v * w[e] : v);
        }
    }
}

// The forms of a head that are read as they lie: d / 8 = LPH lanes of eight values, whole pieces of the rotated part.  Workgroup = (token, some of its
// heads): it forms the angles' sines and cosines once, for all of them, and leaves them with the weights in LDS; a lane asks for its own eight
// values and (pairs half a head apart) for its partners', which a neighbour has too, out of L1: no exchange.  Bound by memory: 2048 tokens of 32 + 2 x 8
// heads of 128 in bf16, 50 MB, 14 us (3.6 TB/s; a wave per head and value by value 39).
template <bool F32>
__device__ __forceinline__ void ld8(const void* base, int64_t at, float (&v)[8]) {
    if constexpr (F32) {
        const f32x4_t a = *reinterpret_cast<const f32x4_t*>((const float*)base + at), b = *reinterpret_cast<const f32x4_t*>((const float*)base + at + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
    } else {
        const uint4 w = ld16((const uint16_t*)base + at);
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[2 * i] = bf16_lo(u[i]), v[2 * i + 1] = bf16_hi(u[i]);
    }
}
template <bool F32>
__device__ __forceinline__ void st8(void* base, int64_t at, const float (&v)[8]) {
    if constexpr (F32) {
        *reinterpret_cast<f32x4_t*>((float*)base + at) = (f32x4_t){v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4_t*>((float*)base + at + 4) = (f32x4_t){v[4], v[5], v[6], v[7]};
    } else {
        st16((uint16_t*)base + at, make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])));
    }
}

template <bool SF32, bool DF32, int LPH>
__global__ __launch_bounds__(256) void slot_store_kernel(SlotStoreArgs a, int heads_per_wg) {
    constexpr int D = LPH * 8, HP = 256 / LPH;
    __shared__ __attribute__((aligned(16))) float wL[2][D], csL[D / 2], snL[D / 2];
    const int units = a.hq + 2 * a.hkv, groups = (units + heads_per_wg - 1) / heads_per_wg, tid = threadIdx.x, half = a.rot / 2;
    const int64_t t = blockIdx.x / groups;
    const int u0 = (int)(blockIdx.x % groups) * heads_per_wg, u1 = min(u0 + heads_per_wg, units), e = tid % LPH * 8;
    const int64_t slot = a.slots[t];
    const bool turned = e < a.rot, low = e < half;
    const int partner = a.adjacent || !turned ? e : low ? e + half : e - half;
    const int64_t row = t * a.ld;
    float x[8], y[8];
    auto fetch = [&](int u) {
        const int h = min(u, units - 1);
        ld8<SF32>(a.qkv, row + (int64_t)h * D + e, x);
        ld8<SF32>(a.qkv, row + (int64_t)h * D + partner, y);
    };
    fetch(u0 + tid / LPH);
    for (int i = tid; i < half; i += 256) {
        float sn, cs;
        sincos_turn(a.positions[t], a.inv_freq[i], sn, cs);
        csL[i] = cs;
        snL[i] = sn;
    }
    for (int i = tid; i < D; i += 256) {
        wL[0][i] = a.q_norm ? a.q_norm[i] : 1.f;
        wL[1][i] = a.k_norm ? a.k_norm[i] : 1.f;
    }
    __syncthreads();
    for (int first = u0; first < u1; first += HP) {       // (the same trips for every lane: exchanges below)
        const int u = first + tid / LPH;
        if (first > u0) fetch(u);
        const bool is_q = u < a.hq, is_v = u >= a.hq + a.hkv;
        float o[8];
        if (is_v) {
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = x[i];
        } else {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
            for (int k = 1; k < LPH; k <<= 1) ss += __shfl_xor(ss, k, 64);      // (a head's lanes go the same way)
            const float inv = (is_q ? a.q_norm : a.k_norm) ? 1.0f / sqrtf(ss / (float)D + a.eps) : 1.f;
            const float* w = wL[is_q ? 0 : 1];
            float xw[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) xw[i] = x[i] * inv * w[e + i];
            if (!turned) {
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = xw[i];
            } else if (a.adjacent) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float cs = csL[e / 2 + i], sn = snL[e / 2 + i];
                    o[2 * i] = xw[2 * i] * cs - xw[2 * i + 1] * sn;
                    o[2 * i + 1] = xw[2 * i + 1] * cs + xw[2 * i] * sn;
                }
            } else {
                const int at = low ? e : e - half;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float yw = y[i] * inv * w[partner + i], sn = snL[at + i];
                    o[i] = xw[i] * csL[at + i] + yw * (low ? -sn : sn);
                }
            }
        }
        if (u >= u1) continue;
        if (is_q) {
            st8<DF32>(a.q_out, t * a.ldq + (int64_t)u * D + e, o);
        } else if (slot >= 0 && slot < a.slots_n) {
            st8<DF32>(is_v ? a.v_cache : a.k_cache, (slot * a.hkv + (u - a.hq - (is_v ? a.hkv : 0))) * D + e, o);
        }
    }
}

// ------------------------------------------------------------------ accept

constexpr int kAcceptLayers = 64;      // layers of one launch: their addresses travel in its arguments
struct AcceptArgs {
    const int64_t *tokens, *picks;
    const int32_t *parents, *row_start, *ctx, *taken, *block_table;
    int64_t bt_stride;
    int bt_cols, rows, n_tokens, max_nodes, max_path, layers, page, num_pages;
    int row_vecs;                      // 16-byte pieces of one token's keys in a layer
    int64_t* ids;
    int32_t *path, *counts, *lens;     // NULL behind the first launch
    u32x4_t* cache[2 * kAcceptLayers];   // keys of the layers, then values
};

// Workgroup = (row, 256 of its pieces: a piece is 16 bytes of a token's keys or values in a layer).  Each workgroup walks for itself:
// the walk is a handful of steps over what fits a wave (n nodes in registers, the picks in LDS), a hand-over from a launch of its own
// would be longer.  A path only ever leads to later nodes (path[j] >= j), so with the moves in order no source has been written.
__global__ __launch_bounds__(256) void tree_accept_kernel(AcceptArgs a) {
    __shared__ int64_t pickL[kTreeNodes];
    __shared__ int pathL[kTreeNodes];
    __shared__ int64_t srcL[kTreeNodes], dstL[kTreeNodes];
    __shared__ int countL;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    TreeRow row = tree_row(a.row_start, b, a.n_tokens, a.max_nodes);
    if (a.taken && a.taken[b] < 0) row.n = 0;      // its nodes were stored nowhere
    const int64_t ctx = max(a.ctx[b], 0);
    if (tid < row.n) pickL[tid] = a.picks[row.start + tid];
    __syncthreads();
    if (wid == 0) {
        int64_t tok[kTreeWords];
        int par[kTreeWords];
#pragma unroll
        for (int w = 0; w < kTreeWords; ++w) {
            const int i = 64 * w + lane;
            par[w] = -2;
            tok[w] = 0;
            if (i < row.n) {
                tok[w] = a.tokens[row.start + i];
                par[w] = a.parents ? a.parents[row.start + i] : i - 1;
            }
        }
        int cur = 0, count = 0;
        while (count < a.max_path && cur < row.n) {
            if (lane == 0) pathL[count] = cur;
            ++count;
            const int64_t pick = pickL[cur];
            int next = row.n;
#pragma unroll
            for (int w = kTreeWords - 1; w >= 0; --w) {
                const uint64_t hit = __builtin_amdgcn_ballot_w64(par[w] == cur && tok[w] == pick && 64 * w + lane > cur);
                if (hit) next = 64 * w + __builtin_ctzll(hit);
            }
            cur = next;
        }
        if (lane == 0) countL = count;
    }
    __syncthreads();
    const int count = countL;
    if (a.counts && blockIdx.y == 0) {
        if (tid == 0) {
            a.counts[b] = count;
            if (a.lens) a.lens[b] = (int)(ctx + count);
        }
        for (int j = tid; j < a.max_path; j += 256) {
            const int node = j < count ? pathL[j] : -1;
            a.path[(int64_t)b * a.max_path + j] = node;
            a.ids[(int64_t)b * a.max_path + j] = node >= 0 ? pickL[node] : -1;
        }
    }
    if (a.layers == 0) return;
    if (tid < count) {
        auto place = [&](int64_t at) -> int64_t {
            const int64_t col = at / a.page;
            if (col >= a.bt_cols) return -1;
            const int pg = a.block_table[(int64_t)b * a.bt_stride + col];
            return pg >= 0 && pg < a.num_pages ? ((int64_t)pg * a.page + at % a.page) * a.row_vecs : -1;
        };
        const int64_t s = place(ctx + pathL[tid]), e = place(ctx + tid);
        srcL[tid] = s;
        dstL[tid] = s < 0 || pathL[tid] == tid ? -1 : e;
    }
    __syncthreads();
    const int64_t item = (int64_t)blockIdx.y * 256 + tid;
    if (item >= (int64_t)2 * a.layers * a.row_vecs) return;
    const int which = (int)(item / a.row_vecs), vec = (int)(item % a.row_vecs);
    u32x4_t* cache = a.cache[which < a.layers ? which : kAcceptLayers + which - a.layers] + vec;
    // eight moves at a time, all read before the first is written: sources lie behind every place that was written in front of them
    for (int first = 0; first < count; first += 8) {
        u32x4_t v[8];
        int64_t to[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            to[i] = first + i < count ? dstL[first + i] : -1;
            if (to[i] >= 0) v[i] = cache[srcL[first + i]];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (to[i] >= 0) cache[to[i]] = v[i];
    }
}

}  // namespace mv

extern "C" {

int mv_tree_plan(const int32_t* ctx_lens, const int32_t* row_start, const int32_t* parents, int32_t* block_table, int64_t bt_stride,
                 int bt_cols, const int32_t* free_pages, int n_free, int rows, int tokens, int max_nodes, int page, int num_pages,
                 int32_t* slots, int32_t* positions, int32_t* row_of, uint64_t* mask, int words, int32_t* taken, mv_stream_t stream) {
    using namespace mv;
    if (rows < 0 || tokens < 0 || max_nodes < 0 || page <= 0 || num_pages <= 0 || bt_cols < 0 || bt_stride < bt_cols || n_free < 0)
        return MV_ERR_INVALID_ARG;
    if ((int64_t)page * num_pages > 0x7fffffff) return MV_ERR_UNSUPPORTED;
    if (rows == 0) return MV_OK;
    if (!ctx_lens || !row_start || !block_table || (n_free > 0 && !free_pages) || !taken ||
        (tokens > 0 && (!slots || !positions || !row_of)))
        return MV_ERR_INVALID_ARG;
    const bool tree = parents || mask;
    if (tree && max_nodes > kTreeNodes) return MV_ERR_UNSUPPORTED;
    if (mask && (words < 1 || words > kTreeWords || words * 64 < max_nodes)) return MV_ERR_INVALID_ARG;
    PlanArgs a{ctx_lens, row_start, parents, free_pages, block_table, bt_stride, bt_cols, n_free, rows, tokens, max_nodes, page,
               num_pages, mask ? words : (max_nodes + 63) / 64, slots, positions, row_of, taken, mask};
    const int threads = tree && max_nodes <= 64 && rows <= 1024 ? 64 : 256;
    const int chunks = tree || max_nodes == 0 ? 1 : (max_nodes + threads - 1) / threads;
    if (chunks > 65535) return MV_ERR_UNSUPPORTED;
    // (a row's workgroup reads the lengths of those before it, whose workgroups write)
    const int64_t r4 = (int64_t)rows * 4, n4 = (int64_t)tokens * 4;
    const MemSpan outs[] = {{slots, n4}, {positions, n4}, {row_of, n4}, {mask, 2 * n4 * words}, {taken, r4}};
    const MemSpan ins[] = {{ctx_lens, r4}, {row_start, r4 + 4}, {parents, n4}, {free_pages, (int64_t)n_free * 4}};
    if (outputs_meet(outs, ins)) return MV_ERR_INVALID_ARG;
    auto in_table = [&](const MemSpan& s) { return rows_meet_span(block_table, bt_stride * 4, (int64_t)bt_cols * 4, rows, s.p, s.n); };
    for (const MemSpan& s : outs)
        if (in_table(s)) return MV_ERR_INVALID_ARG;
    for (const MemSpan& s : ins)
        if (in_table(s)) return MV_ERR_INVALID_ARG;
    hipLaunchKernelGGL(tree_plan_kernel, dim3((unsigned)rows, (unsigned)chunks), dim3((unsigned)threads), 0, (hipStream_t)stream, a);
    return check_launch();
}

int mv_qkv_norm_rotary_slots(const void* qkv, int64_t ld, const float* q_norm, const float* k_norm, float eps, const double* inv_freq,
                             int rot, int adjacent, const int32_t* positions, const int32_t* slots, void* q_out, int64_t ldq,
                             void* k_cache, void* v_cache, int64_t cache_slots, int tokens, int heads, int kv_heads, int d, int src_f32,
                             int dst_f32, mv_stream_t stream) {
    using namespace mv;
    if (tokens < 0 || heads <= 0 || kv_heads <= 0 || d <= 0 || rot < 0 || rot > d || rot % 2 || cache_slots <= 0) return MV_ERR_INVALID_ARG;
    if (src_f32 == 0 && dst_f32) return MV_ERR_UNSUPPORTED;
    if (tokens == 0) return MV_OK;
    if (!qkv || !positions || !slots || !q_out || !k_cache || !v_cache || (rot > 0 && !inv_freq) ||
        ld < (int64_t)(heads + 2 * kv_heads) * d || ldq < (int64_t)heads * d)
        return MV_ERR_INVALID_ARG;
    const int64_t sb = src_f32 ? 4 : 2, db = dst_f32 ? 4 : 2;      // q over its own part of the rows, or nowhere in them
    if (!(q_out == qkv && ld * sb == ldq * db && sb == db) &&
        rows_meet(qkv, ld * sb, (int64_t)(heads + 2 * kv_heads) * d * sb, q_out, ldq * db, (int64_t)heads * d * db, tokens))
        return MV_ERR_INVALID_ARG;
    // nor may the caches, which tokens in any order write, meet each other, q's place or what is read
    const int64_t pool = cache_slots * kv_heads * d * db, t4 = (int64_t)tokens * 4;
    const MemSpan outs[] = {{k_cache, pool}, {v_cache, pool}};
    const MemSpan ins[] = {{positions, t4}, {slots, t4}, {q_norm, d * 4}, {k_norm, d * 4}, {rot > 0 ? inv_freq : nullptr, rot * 4}};
    if (outputs_meet(outs, ins)) return MV_ERR_INVALID_ARG;
    for (const MemSpan& s : outs)
        if (rows_meet_span(qkv, ld * sb, (int64_t)(heads + 2 * kv_heads) * d * sb, tokens, s.p, s.n) ||
            rows_meet_span(q_out, ldq * db, (int64_t)heads * d * db, tokens, s.p, s.n))
            return MV_ERR_INVALID_ARG;
    for (const MemSpan& s : ins)
        if (rows_meet_span(q_out, ldq * db, (int64_t)heads * d * db, tokens, s.p, s.n)) return MV_ERR_INVALID_ARG;
    SlotStoreArgs a{qkv, ld, q_norm, k_norm, eps, inv_freq, rot, adjacent, positions, slots, q_out, ldq, k_cache, v_cache, tokens, heads,
                    kv_heads, d, cache_slots};
    hipStream_t s = (hipStream_t)stream;
    const int units = heads + 2 * kv_heads, sv = src_f32 ? 4 : 8, dv = dst_f32 ? 4 : 8;
    const bool pieces = (d == 64 || d == 128 || d == 256) && rot % (adjacent ? 8 : 16) == 0 && ld % sv == 0 && ldq % dv == 0 && aligned16(qkv) &&
                        aligned16(q_out) && aligned16(k_cache) && aligned16(v_cache);
    if (pieces) {
        // a token's heads in one workgroup where there are tokens for the chip, else in as many as there are rounds of 256 lanes
        const int round = 256 / (d / 8), hpw = tokens >= 4 * num_cus() ? (units + round - 1) / round * round : round;
        const int64_t blocks = (int64_t)tokens * ((units + hpw - 1) / hpw);
        if (blocks > 0x7fffffff) return MV_ERR_UNSUPPORTED;
        const dim3 grid((unsigned)blocks);
#define MV_STORE(S_, D_)                                                                                                      \
    do {                                                                                                                     \
        if (d == 64) hipLaunchKernelGGL((slot_store_kernel<S_, D_, 8>), grid, dim3(256), 0, s, a, hpw);                         \
        else if (d == 128) hipLaunchKernelGGL((slot_store_kernel<S_, D_, 16>), grid, dim3(256), 0, s, a, hpw);                  \
        else hipLaunchKernelGGL((slot_store_kernel<S_, D_, 32>), grid, dim3(256), 0, s, a, hpw);                               \
    } while (0)
        if (src_f32 && dst_f32) MV_STORE(true, true);
        else if (src_f32) MV_STORE(true, false);
        else MV_STORE(false, false);
#undef MV_STORE
        return check_launch();
    }
    const int64_t blocks = ((int64_t)tokens * units + 3) / 4;
    if (blocks > 0x7fffffff) return MV_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)blocks);
    if (src_f32 && dst_f32) hipLaunchKernelGGL((slot_store_any_kernel<true, true>), grid, dim3(256), 0, s, a);
    else if (src_f32) hipLaunchKernelGGL((slot_store_any_kernel<true, false>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((slot_store_any_kernel<false, false>), grid, dim3(256), 0, s, a);
    return check_launch();
}

int mv_tree_accept_planned(const int64_t* tokens, const int64_t* picks, const int32_t* parents, const int32_t* row_start,
                           const int32_t* ctx_lens, const int32_t* taken, const int32_t* block_table, int64_t bt_stride, int bt_cols,
                           void* const* k_caches, void* const* v_caches, int layers, int64_t row_bytes, int page, int num_pages, int rows,
                           int n_tokens, int max_nodes, int max_path, int32_t* path, int64_t* ids, int32_t* counts, int32_t* lens,
                           mv_stream_t stream) {
    using namespace mv;
    if (rows < 0 || n_tokens < 0 || max_nodes < 0 || max_path <= 0 || layers < 0) return MV_ERR_INVALID_ARG;
    if (max_nodes > kTreeNodes || max_path > kTreeNodes) return MV_ERR_UNSUPPORTED;
    if (rows == 0) return MV_OK;
    if (!row_start || !ctx_lens || !path || !ids || !counts || (n_tokens > 0 && (!tokens || !picks))) return MV_ERR_INVALID_ARG;
    AcceptArgs a{tokens, picks, parents, row_start, ctx_lens, taken, block_table, bt_stride, bt_cols, rows, n_tokens, max_nodes, max_path, 0,
                 page, num_pages, 0, ids, path, counts, lens, {}};
    if (layers > 0) {
        if (!block_table || !k_caches || !v_caches || bt_cols < 0 || bt_stride < bt_cols || page <= 0 || num_pages <= 0 || row_bytes <= 0)
            return MV_ERR_INVALID_ARG;
        if (row_bytes % 16 || row_bytes > (1 << 30)) return MV_ERR_UNSUPPORTED;
        for (int i = 0; i < layers; ++i)
            if (!k_caches[i] || !v_caches[i] || !aligned16(k_caches[i]) || !aligned16(v_caches[i])) return MV_ERR_INVALID_ARG;
        a.row_vecs = (int)(row_bytes / 16);
    }
    // (workgroups and launches behind the first still read what the call takes while the outputs are written)
    const int64_t r4 = (int64_t)rows * 4, n4 = (int64_t)n_tokens * 4;
    const MemSpan outs[] = {{path, r4 * max_path}, {ids, 2 * r4 * max_path}, {counts, r4}, {lens, r4}};
    const MemSpan ins[] = {{tokens, 2 * n4}, {picks, 2 * n4}, {parents, n4}, {row_start, r4 + 4}, {ctx_lens, r4}, {taken, r4}};
    if (outputs_meet(outs, ins)) return MV_ERR_INVALID_ARG;
    for (const MemSpan& o : outs)
        if (layers > 0 && rows_meet_span(block_table, bt_stride * 4, (int64_t)bt_cols * 4, rows, o.p, o.n)) return MV_ERR_INVALID_ARG;
    for (int first = 0; first == 0 || first < layers; first += kAcceptLayers) {
        a.layers = layers - first < kAcceptLayers ? layers - first : kAcceptLayers;
        for (int i = 0; i < a.layers; ++i) {
            a.cache[i] = (u32x4_t*)k_caches[first + i];
            a.cache[kAcceptLayers + i] = (u32x4_t*)v_caches[first + i];
        }
        const int64_t items = (int64_t)2 * a.layers * a.row_vecs, parts = items > 0 ? (items + 255) / 256 : 1;
        if (parts > 65535) return MV_ERR_UNSUPPORTED;
        hipLaunchKernelGGL(tree_accept_kernel, dim3((unsigned)rows, (unsigned)parts), dim3(256), 0, (hipStream_t)stream, a);
        const int rc = check_launch();
        if (rc != MV_OK) return rc;
        a.counts = nullptr;
    }
    return MV_OK;
}

int mv_tree_accept(const int64_t* tokens, const int64_t* picks, const int32_t* parents, const int32_t* row_start, const int32_t* ctx_lens,
                   const int32_t* block_table, int64_t bt_stride, int bt_cols, void* const* k_caches, void* const* v_caches, int layers,
                   int64_t row_bytes, int page, int num_pages, int rows, int n_tokens, int max_nodes, int max_path, int32_t* path,
                   int64_t* ids, int32_t* counts, int32_t* lens, mv_stream_t stream) {
    return mv_tree_accept_planned(tokens, picks, parents, row_start, ctx_lens, nullptr, block_table, bt_stride, bt_cols, k_caches, v_caches,
                                  layers, row_bytes, page, num_pages, rows, n_tokens, max_nodes, max_path, path, ids, counts, lens, stream);
}

}  // extern "C"
