// Attention for trees of drafted tokens over the paged cache: node i of row b (tree_ops.hip) sees the row's ctx cached tokens and
// the nodes whose bits its mask has, o = sum_j softmax_j(q . k_j scale) v_j.  The nodes' own keys and values are in the cache already.
//
// The g query heads that share a key/value head are stacked: stacked row r = node * g + head, so every key read serves n * g rows.
// Workgroup = (row, key/value head, run of stacked rows, split of the keys).  Waves take 16-key blocks of the split in turn and
// keep a softmax state each; the states meet in LDS, the splits' in a second launch that adds them in order.
#include "common.h"

namespace mv {

constexpr float kTreeNegBig = -1.0e30f;        // a running maximum before any visible key
constexpr int kTreeMaxNodes = 256;
constexpr int kTreeMaxWords = kTreeMaxNodes / 64;
constexpr int kTreeBlock = 16;                 // keys of a block: pages hold whole blocks

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
    float scale_log2;
};

struct TreeSpan {
    int start, n, ctx, total;    // first token, nodes, cached tokens, keys that have a place in the table
};
__device__ __forceinline__ TreeSpan tree_span(const TreeArgs& a, int b) {
    TreeSpan s;
    s.start = min(max(a.row_start[b], 0), a.tokens);
    s.n = min(min(max(a.row_start[b + 1], s.start), a.tokens) - s.start, a.max_nodes);
    s.ctx = max(a.ctx[b], 0);
    s.total = (int)min((int64_t)s.ctx + s.n, (int64_t)a.bt_cols << a.page_shift);
    return s;
}
// Blocks of a split: all splits of a row but the last take as many, and none fewer than a block a wave
__device__ __forceinline__ int split_blocks(const TreeArgs& a, int total) {
    const int blocks = (total + kTreeBlock - 1) / kTreeBlock;
    return max((blocks + a.nsplit - 1) / a.nsplit, 4);
}
__device__ __forceinline__ int filled_splits_tree(const TreeArgs& a, int total) {
    const int per = split_blocks(a, total), blocks = (total + kTreeBlock - 1) / kTreeBlock;
    return (blocks + per - 1) / per;
}
// 64 bits of a node's mask from bit `first` (negative: cached tokens in front of the nodes, visible) on
__device__ __forceinline__ uint64_t mask_from(const uint64_t (&w)[kTreeMaxWords], int first) {
    if (first <= -64) return ~0ull;
    if (first < 0) return (w[0] << -first) | ((1ull << -first) - 1);
    uint64_t lo = 0, hi = 0;
    const int at = first >> 6, sh = first & 63;
#pragma unroll
    for (int i = 0; i < kTreeMaxWords; ++i) {
        if (i == at) lo = w[i];
        if (i == at + 1) hi = w[i];
    }
    return sh ? (lo >> sh) | (hi << (64 - sh)) : lo;
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

// Both products on v_mfma_f32_16x16x4_f32 (operand A lane (r, q) = A[r][slot q], B likewise, result lane (r, q) = C[4 q + j][r]); the
// contraction's slots are labels.  S^T = K . Q^T: slot q of step j of a group of 16 dimensions is dimension 4 q + j, so a key's and a
// query's values are read 16 (8) bytes a lane.  O^T = V^T . P^T: slot q of step j is key 4 q + j, which is where S^T left its score;
// row r of output block c is dimension 64 h + 4 r + c, so a value row too is read as it lies.  Nothing goes through LDS until the end.
template <bool F32, int D>
__global__ __launch_bounds__(256) void tree_attn_f32_kernel(TreeArgs a) {
    typedef TreeT<F32> X;
    typedef typename X::T T;
    constexpr int RT = 2, W = 4, KG = D / 16, H = D / 64;
    __shared__ __attribute__((aligned(16))) float oL[W][RT * 16][D];
    __shared__ float mL[W][RT * 16], lL[W][RT * 16];
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
    const int split = blockIdx.x % a.nsplit, rest = blockIdx.x / a.nsplit;
    const int rb = rest % a.row_blocks, bh = rest / a.row_blocks, kvh = bh % a.hkv, b = bh / a.hkv;
    const TreeSpan s = tree_span(a, b);
    const int stacked = s.n * a.g, row0 = rb * RT * 16;
    const int per = split_blocks(a, s.total), blocks = (s.total + kTreeBlock - 1) / kTreeBlock;
    const int blk0 = split * per, blk1 = min(blk0 + per, blocks);
    if (row0 >= stacked || (blk0 >= blk1 && split > 0)) return;

    f32x4_t qf[RT][KG];
    uint64_t words[RT][kTreeMaxWords];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int sr = min(row0 + i * 16 + r, stacked - 1), node = sr / a.g;
        const T* qp = (const T*)a.q + (int64_t)(s.start + node) * a.ldq + (int64_t)(kvh * a.g + sr % a.g) * D + 4 * q;
#pragma unroll
        for (int k = 0; k < KG; ++k) qf[i][k] = X::ld4(qp + 16 * k);
#pragma unroll
        for (int w = 0; w < kTreeMaxWords; ++w) {
            if (a.mask) {
                words[i][w] = w < a.words ? a.mask[(int64_t)(s.start + node) * a.words + w] : 0;
            } else {
                const int up = node + 1 - 64 * w;
                words[i][w] = up >= 64 ? ~0ull : up > 0 ? (1ull << up) - 1 : 0;
            }
        }
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
    const int64_t stride = (int64_t)a.hkv * D;
    for (int blk = blk0 + wid; blk < blk1; blk += W) {
        const int kb = blk * kTreeBlock, pg = a.block_table[(int64_t)b * a.bt_stride + (kb >> a.page_shift)];
        if (pg < 0 || pg >= a.num_pages) continue;      // a place without a page: its keys do not count
        const int64_t row = ((int64_t)pg << a.page_shift) + (kb & (a.page - 1));
        const T* kp = (const T*)a.k_cache + (row + r) * stride + (int64_t)kvh * D + 4 * q;
        const T* vp = (const T*)a.v_cache + (row + 4 * q) * stride + (int64_t)kvh * D + 4 * r;
        f32x4_t kf[KG], vf[4][H];
#pragma unroll
        for (int k = 0; k < KG; ++k) kf[k] = X::ld4(kp + 16 * k);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int h = 0; h < H; ++h) vf[j][h] = X::ld4(vp + j * stride + 64 * h);
        const bool open = kb + kTreeBlock <= s.ctx;      // every key visible to every row (uniform)
        // Where a row may not see a key, its weight is zero and the product would still hand on a value that is not finite: such
        // values are left out of the product and added by hand to the rows that do see them; behind the last key everything is.
        bool odd = false;
        if (!open) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        if (kb + 4 * q + j >= s.total) vf[j][h][c] = 0.f;
                        if (!(fabsf(vf[j][h][c]) <= 3.4028235e38f)) {
                            vf[j][h][c] = 0.f;
                            odd = true;
                        }
                    }
            odd = __builtin_amdgcn_ballot_w64(odd) != 0;
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            if (row0 + i * 16 >= stacked) break;         // uniform
            f32x4_t sc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < KG; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j) sc = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[k][j], qf[i][k][j], sc, 0, 0, 0);
            uint32_t seen = 0xffff;
            if (!open) {
                seen = (uint32_t)mask_from(words[i], kb - s.ctx);
                if (s.total - kb < 16) seen &= (1u << (s.total - kb)) - 1;
                seen &= 0xffff;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (!(seen >> (4 * q + j) & 1)) sc[j] = -__builtin_inff();
            }
            float top = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])) * a.scale_log2;
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float mn = fmaxf(m[i], top), alpha = __builtin_amdgcn_exp2f(m[i] - mn);
            m[i] = mn;
            f32x4_t p;
#pragma unroll
            for (int j = 0; j < 4; ++j) p[j] = __builtin_amdgcn_exp2f(fmaf(sc[j], a.scale_log2, -mn));
            l[i] = l[i] * alpha + ((p[0] + p[1]) + (p[2] + p[3]));
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    acc[i][h][c] *= alpha;
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][h][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[j][h][c], p[j], acc[i][h][c], 0, 0, 0);
                }
            if (odd) {
                for (int key = 0; key < 16 && kb + key < s.total; ++key) {
                    float pk = 0.f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float v = __shfl(p[j], (key >> 2) * 16 + r, 64);
                        if ((key & 3) == j) pk = v;
                    }
                    if (!(seen >> key & 1)) continue;
                    const T* v = (const T*)a.v_cache + (row + key) * stride + (int64_t)kvh * D;
#pragma unroll
                    for (int h = 0; h < H; ++h)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const f32x4_t x = X::ld4(v + 64 * h + 16 * q + 4 * e);
#pragma unroll
                            for (int c = 0; c < 4; ++c)
                                if (!(fabsf(x[c]) <= 3.4028235e38f)) acc[i][h][c][e] += pk * x[c];
                        }
                }
            }
        }
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
    __syncthreads();
    const bool whole = filled_splits_tree(a, s.total) <= 1;
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
        const int64_t t = s.start + sr / a.g;
        const int head = kvh * a.g + sr % a.g;
        if (whole) {
            const float inv = den != 0.f ? 1.0f / den : 0.f;      // nothing visible: zeros
            X::st4((T*)a.out + t * a.ldo + (int64_t)head * D + c, o * inv);
        } else {
            const int64_t at = ((int64_t)split * a.tokens + t) * a.hq + head;
            *reinterpret_cast<f32x4_t*>(a.part + at * D + c) = o;
            if (c == 0) {
                a.state[2 * at] = top;
                a.state[2 * at + 1] = den;
            }
        }
    }
}

// Splits added in order; rows that one split holds are written already.
template <bool F32, int D>
__global__ __launch_bounds__(256) void tree_attn_merge_kernel(TreeArgs a) {
    typedef TreeT<F32> X;
    constexpr int LPR = D / 4;                 // lanes of a (node, head)
    const int b = blockIdx.y;
    const TreeSpan s = tree_span(a, b);
    const int filled = filled_splits_tree(a, s.total);
    const int64_t item = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
    const int node = (int)(item / a.hq), head = (int)(item % a.hq), c = threadIdx.x % LPR * 4;
    if (filled <= 1 || node >= s.n) return;
    const int64_t t = s.start + node, step = (int64_t)a.tokens * a.hq, at = t * a.hq + head;
    float top = kTreeNegBig;
    for (int i = 0; i < filled; ++i) top = fmaxf(top, a.state[2 * (at + i * step)]);
    float den = 0.f;
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < filled; ++i) {
        const float f = __builtin_amdgcn_exp2f(a.state[2 * (at + i * step)] - top);
        den = fmaf(a.state[2 * (at + i * step) + 1], f, den);
        o += *reinterpret_cast<const f32x4_t*>(a.part + (at + i * step) * D + c) * f;
    }
    const float inv = den != 0.f ? 1.0f / den : 0.f;
    X::st4((typename X::T*)a.out + t * a.ldo + (int64_t)head * D + c, o * inv);
}

}  // namespace mv

extern "C" {

size_t mv_tree_attn_workspace_bytes(int tokens, int hq, int d, int num_splits) {
    if (tokens <= 0 || hq <= 0 || d <= 0 || num_splits <= 1) return 0;
    return (size_t)num_splits * tokens * hq * (d + 2) * sizeof(float);
}

int mv_tree_attn_pick_splits(int rows, int max_nodes, int hq, int hkv, int d, int max_keys) {
    if (rows <= 0 || max_nodes <= 0 || hq <= 0 || hkv <= 0 || max_keys <= 0) return 1;
    const int64_t row_blocks = ((int64_t)max_nodes * (hq / hkv) + 31) / 32, units = rows * (int64_t)hkv * row_blocks;
    int64_t splits = (2 * mv::num_cus() + units - 1) / units;
    const int64_t most = ((int64_t)max_keys + 63) / 64;
    if (splits > most) splits = most;
    return (int)(splits < 1 ? 1 : splits > 64 ? 64 : splits);
}

int mv_tree_attn(const void* q, int64_t ldq, const void* k_cache, const void* v_cache, const int32_t* ctx_lens, const int32_t* row_start,
                 const int32_t* block_table, int64_t bt_stride, int bt_cols, const uint64_t* mask, int words, void* out, int64_t ldo,
                 void* workspace, size_t workspace_bytes, int rows, int tokens, int max_nodes, int hq, int hkv, int d, int page,
                 int num_pages, float scale, int num_splits, int f32, mv_stream_t stream) {
    using namespace mv;
    if (rows < 0 || tokens < 0 || max_nodes < 0 || hq <= 0 || hkv <= 0 || hq % hkv || page <= 0 || num_pages <= 0 || bt_cols <= 0 ||
        bt_stride < bt_cols || num_splits < 1 || !(scale > 0.f) || scale > 3.0e38f)
        return MV_ERR_INVALID_ARG;
    if ((d != 64 && d != 128) || hq / hkv > 8 || (page & (page - 1)) || page < kTreeBlock || max_nodes > kTreeMaxNodes || num_splits > 64)
        return MV_ERR_UNSUPPORTED;
    if (rows == 0 || tokens == 0 || max_nodes == 0) return MV_OK;
    if (!q || !k_cache || !v_cache || !ctx_lens || !row_start || !block_table || !out) return MV_ERR_INVALID_ARG;
    if (mask && (words < 1 || words > kTreeMaxWords || words * 64 < max_nodes)) return MV_ERR_INVALID_ARG;
    const int vec = f32 ? 4 : 8;
    if (ldq < (int64_t)hq * d || ldo < (int64_t)hq * d || ldq % vec || ldo % vec || !aligned16(q) || !aligned16(out) ||
        !aligned16(k_cache) || !aligned16(v_cache))
        return MV_ERR_INVALID_ARG;
    if (num_splits > 1 && (!workspace || !aligned16(workspace) || workspace_bytes < mv_tree_attn_workspace_bytes(tokens, hq, d, num_splits)))
        return MV_ERR_WORKSPACE;
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
    a.row_blocks = (max_nodes * a.g + 31) / 32;
    a.scale_log2 = scale * 1.4426950408889634f;
    const int64_t grid = (int64_t)rows * hkv * a.row_blocks * num_splits;
    if (grid > 0x7fffffff || rows > 65535) return MV_ERR_UNSUPPORTED;
    hipStream_t s = (hipStream_t)stream;
    const dim3 g1((unsigned)grid);
#define MV_TREE(F32_, D_)                                                                                                     \
    do {                                                                                                                      \
        hipLaunchKernelGGL((tree_attn_f32_kernel<F32_, D_>), g1, dim3(256), 0, s, a);                                           \
        if (num_splits > 1)                                                                                                   \
            hipLaunchKernelGGL((tree_attn_merge_kernel<F32_, D_>), dim3((unsigned)((max_nodes * hq + 1024 / D_ - 1) / (1024 / D_)), (unsigned)rows), \
                               dim3(256), 0, s, a);                                                                             \
    } while (0)
    if (f32 && d == 64) MV_TREE(true, 64);
    else if (f32) MV_TREE(true, 128);
    else if (d == 64) MV_TREE(false, 64);
    else MV_TREE(false, 128);
#undef MV_TREE
    return check_launch();
}

}  // extern "C"
