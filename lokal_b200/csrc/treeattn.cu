// Attention of drafted rows over a paged cache: lokal_cuda_tree_attn, its plan (lokal_cuda_tree_plan) and the kernel
// that takes every type and shape.
//
// A sequence holds c committed rows and, behind them, n drafted rows (speculative decoding: a tree of candidate
// tokens; n = 1 is plain decoding, a chain is a chunk of a prompt). Drafted row i sees every committed row and the
// drafted rows its mask names:
//   z_t = scale * q_i . k_t ,   out_i = sum_t exp(z_t - max z) v_t / sum_t exp(z_t - max z)   over the visible t
// in one pass over the keys with a running maximum and sum (the accumulated v is rescaled when the maximum grows). A row
// that sees nothing gets zeros. K and V are read once for the query heads that share a key head.
#include "treeattn.cuh"

namespace lokal {
namespace {

// ---- the kernel for any type and shape ----
// All arithmetic in f32, 128 threads, tiles of 16 query rows and 64 keys. K, V and q are widened into shared memory once;
// scores: a thread holds 2 rows x 4 keys (rows padded by four floats, so the 16 keys that a half warp reads at the same
// column lie in different banks); output: a thread holds one or two columns of 8 or 16 rows.
constexpr int kAnyRows = 16, kAnyKeys = 64, kAnyThreads = 128;
constexpr int kScoreStride = 20;  // scores are kept by key, 16 rows each: 16-byte aligned and off the banks of a power of two

template <int HDP>
constexpr size_t any_smem() {
    return (static_cast<size_t>(kAnyRows + kAnyKeys) * (HDP + 4) + static_cast<size_t>(kAnyKeys) * HDP + kAnyKeys * kScoreStride + 3 * kAnyRows) * 4 +
           kAnyKeys * 8 + 16 * 8;
}

template <typename T>
__device__ __forceinline__ void load4(const T* p, bool vec, unsigned left, float (&f)[4]) {
    if (vec && left >= 4) {
        if constexpr (sizeof(T) == 4) {
            const float4 v = *reinterpret_cast<const float4*>(p);
            f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
        } else {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            float t[8];
            unpack16<T>(make_uint4(v.x, v.y, 0u, 0u), t);
            f[0] = t[0], f[1] = t[1], f[2] = t[2], f[3] = t[3];
        }
    } else {
#pragma unroll
        for (unsigned j = 0; j < 4; j++) f[j] = j < left ? to_f32<T>(p[j]) : 0.0f;
    }
}

template <typename TQ, typename TK, int HDP>
__global__ void __launch_bounds__(kAnyThreads) tree_attn_any_kernel(const TreeArgs a, int kv_vec, int q_vec) {
    pdl_sync();
    constexpr int ROWS = HDP == 64 ? 8 : 16, COLS = HDP <= 128 ? 1 : HDP / 128;  // of the output, per thread
    extern __shared__ __align__(16) unsigned char smem[];
    float* qs = reinterpret_cast<float*>(smem);
    float* ks = qs + kAnyRows * (HDP + 4);
    float* vs = ks + kAnyKeys * (HDP + 4);
    float* ps = vs + kAnyKeys * HDP;
    float* row_m = ps + kAnyKeys * kScoreStride;
    float* row_l = row_m + kAnyRows;
    float* row_scale = row_l + kAnyRows;
    unsigned long long* row_at = reinterpret_cast<unsigned long long*>(row_scale + kAnyRows);  // cache row of each key of the tile
    unsigned long long* sh = row_at + kAnyKeys;
    const unsigned tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const unsigned shares = gridDim.x;
    const TreePlace place = tree_locate<kAnyKeys, kAnyThreads>(a, sh, blockIdx.x == 0, [&](unsigned total) {
        const TreeShares s(total, shares);
        return blockIdx.x < s.g ? s.first(blockIdx.x) : total;
    });
    if (place.seq >= a.n_seqs) return;
    const TreeShares share(place.total, shares);
    TreeWalk<kAnyKeys> walk;
    walk.start(a, place, share.first(blockIdx.x), share.first(blockIdx.x + 1));
    TreeUnit u;
    const unsigned hd = a.head_dim;
    while (walk.next(a, u)) {
        const unsigned rows_all = u.seq.n * a.group, flat0 = u.block * kAnyRows;
        const unsigned m_rows = min(static_cast<unsigned>(kAnyRows), rows_all - flat0);
        __syncthreads();  // the unit before may still be read
        for (unsigned e = tid; e < kAnyRows * (HDP / 4); e += kAnyThreads) {
            const unsigned r = e / (HDP / 4), d = (e % (HDP / 4)) * 4;
            float f[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (r < m_rows && d < hd) {
                const unsigned flat = flat0 + r, node = flat / a.group, head = u.kv_head * a.group + flat % a.group;
                const TQ* p = static_cast<const TQ*>(a.q) + static_cast<size_t>(u.seq.row0 + node) * a.q_stride + static_cast<size_t>(head) * hd + d;
                load4<TQ>(p, q_vec, hd - d, f);
            }
            *reinterpret_cast<float4*>(qs + r * (HDP + 4) + d) = make_float4(f[0], f[1], f[2], f[3]);
        }
        if (tid < kAnyRows) {
            row_m[tid] = -INFINITY;
            row_l[tid] = 0.0f;
        }
        float acc[COLS][ROWS];
#pragma unroll
        for (int c = 0; c < COLS; c++)
#pragma unroll
            for (int r = 0; r < ROWS; r++) acc[c][r] = 0.0f;
        const unsigned col = HDP == 64 ? tid & 63u : tid, row0 = HDP == 64 ? (tid >> 6) * 8 : 0u;
        for (unsigned kt = u.k0; kt < u.k1; kt++) {
            const int pos0 = static_cast<int>(kt) * kAnyKeys;
            const unsigned keys = min(static_cast<unsigned>(kAnyKeys), static_cast<unsigned>(u.seq.len - pos0));
            __syncthreads();  // K, V and the scores of the tile before are done with
            if (tid < keys) {
                const unsigned pos = static_cast<unsigned>(pos0) + tid;
                row_at[tid] = (static_cast<unsigned long long>(tree_page(a, u.seq.slot, pos >> a.page_shift)) << a.page_shift) + (pos & (a.page_rows - 1));
            }
            __syncthreads();
            for (unsigned e = tid; e < kAnyKeys * (HDP / 4); e += kAnyThreads) {
                const unsigned key = e / (HDP / 4), d = (e % (HDP / 4)) * 4;
                float fk[4] = {0.0f, 0.0f, 0.0f, 0.0f}, fv[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                if (key < keys && d < hd) {
                    const size_t off = row_at[key] * a.row_bytes + (static_cast<size_t>(u.kv_head) * hd + d) * sizeof(TK);
                    load4<TK>(reinterpret_cast<const TK*>(a.k + off), kv_vec, hd - d, fk);
                    load4<TK>(reinterpret_cast<const TK*>(a.v + off), kv_vec, hd - d, fv);
                }
                *reinterpret_cast<float4*>(ks + key * (HDP + 4) + d) = make_float4(fk[0], fk[1], fk[2], fk[3]);
                *reinterpret_cast<float4*>(vs + key * HDP + d) = make_float4(fv[0], fv[1], fv[2], fv[3]);
            }
            __syncthreads();
            {   // scores
                const unsigned kg = tid & 15u, rg = (tid >> 4) * 2;
                float s[2][4] = {};
                for (unsigned d = 0; d < hd; d += 4) {
                    const float4 q0 = *reinterpret_cast<const float4*>(qs + rg * (HDP + 4) + d);
                    const float4 q1 = *reinterpret_cast<const float4*>(qs + (rg + 1) * (HDP + 4) + d);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float4 k = *reinterpret_cast<const float4*>(ks + (kg + 16 * j) * (HDP + 4) + d);
                        s[0][j] = fmaf(q0.x, k.x, fmaf(q0.y, k.y, fmaf(q0.z, k.z, fmaf(q0.w, k.w, s[0][j]))));
                        s[1][j] = fmaf(q1.x, k.x, fmaf(q1.y, k.y, fmaf(q1.z, k.z, fmaf(q1.w, k.w, s[1][j]))));
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    ps[(kg + 16 * j) * kScoreStride + rg] = s[0][j] * a.scale_log2;
                    ps[(kg + 16 * j) * kScoreStride + rg + 1] = s[1][j] * a.scale_log2;
                }
            }
            __syncthreads();
#pragma unroll
            for (int rr = 0; rr < 4; rr++) {  // a warp has four rows
                const unsigned r = warp * 4 + rr;
                const unsigned node = (flat0 + min(r, m_rows - 1)) / a.group;
                float z[2], m = row_m[r], top;
                bool seen[2];
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const unsigned bits = tree_visible(a, u.seq, node, pos0 + 32 * j);
                    seen[j] = (bits >> lane) & 1u;
                    z[j] = seen[j] ? ps[(lane + 32 * j) * kScoreStride + r] : -INFINITY;
                }
                top = fmaxf(z[0], z[1]);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                top = fmaxf(top, m);
                const float ref = top == -INFINITY ? 0.0f : top;
                // -0 marks a key that is not seen: it adds nothing to the sum, and the product below can tell it from a
                // weight that has become 0
                const float p0 = seen[0] ? exp2f(z[0] - ref) : -0.0f, p1 = seen[1] ? exp2f(z[1] - ref) : -0.0f;
                const float sum = warp_sum(p0 + p1);
                ps[lane * kScoreStride + r] = p0;
                ps[(lane + 32) * kScoreStride + r] = p1;
                __syncwarp();
                if (lane == 0) {
                    const float scale = exp2f(m - ref);  // 0 where nothing was visible before
                    row_scale[r] = scale;
                    row_m[r] = top;
                    row_l[r] = fmaf(row_l[r], scale, sum);
                }
            }
            __syncthreads();
#pragma unroll
            for (int r = 0; r < ROWS; r++) {
                const float scale = row_scale[row0 + r];
#pragma unroll
                for (int c = 0; c < COLS; c++) acc[c][r] *= scale;
            }
            // A drafted row that a query row does not see may hold an infinity or a NaN: in tiles with drafted rows such a
            // key is left out instead of being multiplied by 0.
            const bool drafted = pos0 + static_cast<int>(keys) > u.seq.ctx;
            for (unsigned key = 0; key < keys; key++) {
                float p[ROWS];
#pragma unroll
                for (int r = 0; r < ROWS; r += 4) {
                    const float4 t = *reinterpret_cast<const float4*>(ps + key * kScoreStride + row0 + r);
                    p[r] = t.x, p[r + 1] = t.y, p[r + 2] = t.z, p[r + 3] = t.w;
                }
#pragma unroll
                for (int c = 0; c < COLS; c++) {
                    const float v = vs[key * HDP + col + c * 128];
                    if (drafted) {
#pragma unroll
                        for (int r = 0; r < ROWS; r++) acc[c][r] = __float_as_uint(p[r]) == 0x80000000u ? acc[c][r] : fmaf(p[r], v, acc[c][r]);
                    } else {
#pragma unroll
                        for (int r = 0; r < ROWS; r++) acc[c][r] = fmaf(p[r], v, acc[c][r]);
                    }
                }
            }
        }
        // the block is done, or a piece of it
        if (u.whole) {
#pragma unroll
            for (int r = 0; r < ROWS; r++) {
                const unsigned row = row0 + r;
                if (row >= m_rows) break;
                const unsigned flat = flat0 + row, node = flat / a.group, head = u.kv_head * a.group + flat % a.group;
                TQ* dst = static_cast<TQ*>(a.out) + static_cast<size_t>(u.seq.row0 + node) * a.out_stride + static_cast<size_t>(head) * hd;
                const float l = row_l[row];
#pragma unroll
                for (int c = 0; c < COLS; c++)
                    if (col + c * 128 < hd) dst[col + c * 128] = from_f32<TQ>(l == 0.0f ? 0.0f : acc[c][r] / l);
            }
        } else {
            const size_t slot = (static_cast<size_t>(blockIdx.x) * 2 + u.piece) * kAnyRows;
#pragma unroll
            for (int r = 0; r < ROWS; r++) {
#pragma unroll
                for (int c = 0; c < COLS; c++)
                    if (col + c * 128 < hd) a.part_o[(slot + row0 + r) * hd + col + c * 128] = acc[c][r];
            }
            if (tid < kAnyRows) a.part_ml[slot + tid] = make_float2(row_m[tid], row_l[tid]);
        }
    }
}

// CTAs of the kernel above per SM: what its shared memory allows (41, 79 and 155 KB of 227).
constexpr unsigned any_ctas(unsigned head_dim) { return head_dim <= 64 ? 5 : head_dim <= 128 ? 2 : 1; }

template <typename TQ, typename TK, int HDP>
int launch_any_hd(lokal_cuda_ctx* ctx, cudaStream_t s, const TreeArgs& a, int kv_vec, int q_vec) {
    auto kern = tree_attn_any_kernel<TQ, TK, HDP>;
    constexpr size_t smem = any_smem<HDP>();
    const unsigned shares = static_cast<unsigned>(ctx->sm_count) * any_ctas(a.head_dim);
    launch_staged(kern, shares, kAnyThreads, smem, s, a, kv_vec, q_vec);
    LOKAL_CHECK_LAUNCH(ctx, "tree_attn_any_kernel");
    launch_k(tree_join_kernel<TQ, kAnyRows, kAnyKeys>, shares - 1, 256, 0, s, a, shares);
    LOKAL_CHECK_LAUNCH(ctx, "tree_join_kernel");
    return LOKAL_OK;
}

template <typename TQ, typename TK>
int launch_any(lokal_cuda_ctx* ctx, cudaStream_t s, const TreeArgs& a) {
    const int kv_vec = a.head_dim % 4 == 0 && a.row_bytes % (4 * sizeof(TK)) == 0 && aligned_to(a.k, 4 * sizeof(TK)) && aligned_to(a.v, 4 * sizeof(TK));
    const int q_vec = a.head_dim % 4 == 0 && a.q_stride % 4 == 0 && aligned_to(a.q, 4 * sizeof(TQ));
    if (a.head_dim <= 64) return launch_any_hd<TQ, TK, 64>(ctx, s, a, kv_vec, q_vec);
    if (a.head_dim <= 128) return launch_any_hd<TQ, TK, 128>(ctx, s, a, kv_vec, q_vec);
    return launch_any_hd<TQ, TK, 256>(ctx, s, a, kv_vec, q_vec);
}

template <typename TQ>
int launch_any_q(lokal_cuda_ctx* ctx, cudaStream_t s, const TreeArgs& a, int kv_dtype) {
    switch (kv_dtype) {
        case LOKAL_F32: return launch_any<TQ, float>(ctx, s, a);
        case LOKAL_F16: return launch_any<TQ, __half>(ctx, s, a);
        default: return launch_any<TQ, __nv_bfloat16>(ctx, s, a);
    }
}

size_t any_rows(const lokal_cuda_ctx* ctx, unsigned head_dim) { return static_cast<size_t>(ctx->sm_count) * any_ctas(head_dim) * 2 * kAnyRows; }

// ---- mask, positions and cache rows of drafted trees ----
struct PlanArgs {
    const int32_t* parents;
    unsigned long long* mask;
    int32_t* positions;
    uint32_t* cache_rows;
};

// A CTA per sequence, a thread per drafted row: the row's ancestors are found by following its parents, which come
// before it, so the walk ends. Trees are a few hundred rows at most; the parents stay in L1.
__global__ void __launch_bounds__(128) tree_plan_kernel(const TreeArgs a, const PlanArgs t) {
    pdl_sync();
    const TreeSeq q = tree_seq(a, blockIdx.x, threadIdx.x == 0);
    for (unsigned j = threadIdx.x; j < q.n; j += 128) {
        const size_t row = q.row0 + j;
        unsigned depth = 0;
        bool bad = false;
        if (t.mask) {
            for (unsigned w = 0; w < a.mask_words; w++) t.mask[row * a.mask_words + w] = 0ull;
            if ((j >> 6) >= a.mask_words) bad = true;
        }
        if (!t.parents) {  // a chain
            depth = j + 1;
            for (unsigned w = 0; t.mask && w < a.mask_words && w <= j >> 6; w++) t.mask[row * a.mask_words + w] = w < j >> 6 ? ~0ull : (2ull << (j & 63u)) - 1ull;
        }
        for (int at = t.parents ? static_cast<int>(j) : -1; at >= 0;) {
            if (t.mask && static_cast<unsigned>(at) >> 6 < a.mask_words)
                t.mask[row * a.mask_words + (static_cast<unsigned>(at) >> 6)] |= 1ull << (static_cast<unsigned>(at) & 63u);
            depth++;
            int up = t.parents[q.row0 + static_cast<unsigned>(at)];
            if (up < -1 || up >= at) {
                bad = true;
                up = -1;
            }
            at = up;
        }
        if (bad) atomicOr(a.err_word, kErrPageRange);
        if (t.positions) t.positions[row] = q.ctx + static_cast<int>(depth) - 1;
        if (t.cache_rows) {
            const unsigned pos = static_cast<unsigned>(q.ctx) + j;
            const int page = a.table[static_cast<size_t>(q.slot) * a.max_pages + (pos >> a.page_shift)];
            const bool ok = page >= 0 && static_cast<unsigned>(page) < a.n_pages;
            if (!ok) atomicOr(a.err_word, kErrPosRange);
            t.cache_rows[row] = ok ? (static_cast<unsigned>(page) << a.page_shift) + (pos & (a.page_rows - 1)) : LOKAL_KV_ROW_NONE;
        }
    }
}

TreeArgs tree_args(const lokal_cuda_ctx* ctx, const lokal_kv_pool* pool, const uint32_t* slots, const int32_t* q_start, size_t n_seqs, size_t rows) {
    TreeArgs a{};
    a.slots = slots;
    a.q_start = q_start;
    a.table = pool->a.table;
    a.lens = pool->a.lens;
    a.err_word = ctx->err_word;
    a.row_bytes = pool->a.row_bytes;
    a.n_seqs = static_cast<unsigned>(n_seqs);
    a.rows = static_cast<unsigned>(rows);
    a.page_rows = pool->a.page_rows;
    a.page_shift = pool->a.page_shift;
    a.n_pages = pool->a.n_pages;
    a.n_slots = pool->a.n_slots;
    a.max_pages = pool->a.max_pages;
    return a;
}

}  // namespace
}  // namespace lokal

extern "C" {

int lokal_cuda_tree_plan(lokal_cuda_ctx* ctx, lokal_cuda_stream s, const lokal_kv_pool* pool, const uint32_t* slots, const int32_t* q_start,
                         size_t n_seqs, size_t rows, const int32_t* parents, uint64_t* mask, uint32_t mask_words, int32_t* positions,
                         uint32_t* cache_rows) {
    if (!ctx) return LOKAL_ERR_BAD_ARG;
    lokal::DeviceGuard guard(ctx->device);
    if (!guard.ok) return ctx->fail(LOKAL_ERR_CUDA, "cannot select device %d", ctx->device);
    if (!pool || pool->device != ctx->device) return ctx->fail(LOKAL_ERR_BAD_ARG, "tree_plan: the pool is null or on another device");
    if (n_seqs && !q_start) return ctx->fail(LOKAL_ERR_BAD_ARG, "tree_plan: q_start must be non-null");
    if (mask && mask_words == 0) return ctx->fail(LOKAL_ERR_BAD_ARG, "tree_plan: a mask needs mask_words");
    if (n_seqs > 0x7fffffffull || rows > 0x7fffffffull) return ctx->fail(LOKAL_ERR_BAD_ARG, "tree_plan: too many sequences or rows");
    if (!lokal::aligned_to(q_start, 4) || !lokal::aligned_to(slots, 4) || !lokal::aligned_to(parents, 4) || !lokal::aligned_to(positions, 4) ||
        !lokal::aligned_to(cache_rows, 4) || !lokal::aligned_to(mask, 8))
        return ctx->fail(LOKAL_ERR_MISALIGNED, "tree_plan: a pointer is not aligned to its element size");
    if (n_seqs == 0 || rows == 0) return LOKAL_OK;
    lokal::TreeArgs a = lokal::tree_args(ctx, pool, slots, q_start, n_seqs, rows);
    a.mask_words = mask_words;
    const lokal::PlanArgs t{parents, reinterpret_cast<unsigned long long*>(mask), positions, cache_rows};
    lokal::launch_k(lokal::tree_plan_kernel, static_cast<unsigned>(n_seqs), 128, 0, static_cast<cudaStream_t>(s), a, t);
    LOKAL_CHECK_LAUNCH(ctx, "tree_plan_kernel");
    return LOKAL_OK;
}

size_t lokal_cuda_tree_attn_workspace(const lokal_cuda_ctx* ctx, size_t rows, uint32_t n_q_heads, uint32_t n_kv_heads, uint32_t head_dim) {
    if (!ctx || rows == 0 || n_q_heads == 0 || n_kv_heads == 0 || head_dim == 0 || head_dim > 256) return 0;
    size_t most = lokal::any_rows(ctx, head_dim);
    if (head_dim == 64 || head_dim == 128) {
        const size_t tc = lokal::tree_tc_rows(ctx), mma = lokal::tree_mma_rows(ctx, head_dim);
        if (tc > most) most = tc;
        if (mma > most) most = mma;
    }
    return most * (head_dim + 2) * sizeof(float);
}

int lokal_cuda_tree_attn(lokal_cuda_ctx* ctx, lokal_cuda_stream s, const lokal_kv_pool* pool, uint32_t k_store, uint32_t v_store,
                         const uint32_t* slots, const int32_t* q_start, size_t n_seqs, size_t rows, const uint64_t* mask, uint32_t mask_words,
                         const void* q, size_t q_row_stride, void* out, size_t out_row_stride, uint32_t n_q_heads, uint32_t n_kv_heads,
                         uint32_t head_dim, float scale, int dtype, int kv_dtype, void* workspace, size_t workspace_bytes) {
    if (!ctx) return LOKAL_ERR_BAD_ARG;
    lokal::DeviceGuard guard(ctx->device);
    if (!guard.ok) return ctx->fail(LOKAL_ERR_CUDA, "cannot select device %d", ctx->device);
    if (!pool || pool->device != ctx->device) return ctx->fail(LOKAL_ERR_BAD_ARG, "tree_attn: the pool is null or on another device");
    if (k_store >= pool->a.n_stores || v_store >= pool->a.n_stores)
        return ctx->fail(LOKAL_ERR_BAD_ARG, "tree_attn: stores %u / %u of a pool of %u", k_store, v_store, pool->a.n_stores);
    if (!lokal::is_act_type(dtype) || !lokal::is_act_type(kv_dtype))
        return ctx->fail(LOKAL_ERR_UNSUPPORTED, "tree_attn: types %d / %d are not F32/F16/BF16", dtype, kv_dtype);
    if (n_kv_heads == 0 || n_q_heads == 0 || n_q_heads % n_kv_heads)
        return ctx->fail(LOKAL_ERR_BAD_ARG, "tree_attn: %u query heads do not divide over %u key heads", n_q_heads, n_kv_heads);
    if (head_dim == 0) return ctx->fail(LOKAL_ERR_BAD_ARG, "tree_attn: head_dim is zero");
    if (head_dim > 256) return ctx->fail(LOKAL_ERR_UNSUPPORTED, "tree_attn: head_dim %u is above 256", head_dim);
    const size_t es = lokal::type_size(dtype), ks = lokal::type_size(kv_dtype);
    const uint64_t width = static_cast<uint64_t>(n_q_heads) * head_dim;
    if (static_cast<uint64_t>(n_kv_heads) * head_dim * ks > pool->a.row_bytes)
        return ctx->fail(LOKAL_ERR_BAD_ARG, "tree_attn: a cache row of %zu bytes does not hold %u heads of %u", pool->a.row_bytes, n_kv_heads, head_dim);
    if (pool->a.row_bytes % ks) return ctx->fail(LOKAL_ERR_BAD_ARG, "tree_attn: cache rows of %zu bytes are not whole elements", pool->a.row_bytes);
    if (n_seqs > 0x7fffffffull || rows > 0x7fffffffull || static_cast<uint64_t>(rows) * n_q_heads > 0x7fffffffull)
        return ctx->fail(LOKAL_ERR_BAD_ARG, "tree_attn: too many sequences or rows");
    if (mask && mask_words == 0) return ctx->fail(LOKAL_ERR_BAD_ARG, "tree_attn: a mask needs mask_words");
    if (n_seqs == 0 || rows == 0) return LOKAL_OK;
    if (!q || !out || !q_start) return ctx->fail(LOKAL_ERR_BAD_ARG, "tree_attn: q, out and q_start must be non-null");
    if (q == out) return ctx->fail(LOKAL_ERR_BAD_ARG, "tree_attn: out must not be q");
    if (q_row_stride < width || out_row_stride < width) return ctx->fail(LOKAL_ERR_BAD_ARG, "tree_attn: a row stride is smaller than the heads");
    if (!lokal::aligned_to(q, es) || !lokal::aligned_to(out, es) || !lokal::aligned_to(pool->stores[k_store], ks) || !lokal::aligned_to(pool->stores[v_store], ks) ||
        !lokal::aligned_to(q_start, 4) || !lokal::aligned_to(slots, 4) || !lokal::aligned_to(mask, 8) || !lokal::aligned_to(workspace, 16))
        return ctx->fail(LOKAL_ERR_MISALIGNED, "tree_attn: a pointer is not aligned to its element size (the workspace to 16 bytes)");
    const size_t need = lokal_cuda_tree_attn_workspace(ctx, rows, n_q_heads, n_kv_heads, head_dim);
    if (!workspace || workspace_bytes < need)
        return ctx->fail(LOKAL_ERR_BAD_ARG, "tree_attn: a workspace of %zu bytes is needed, %zu were given", need, workspace ? workspace_bytes : 0);
    lokal::TreeArgs a = lokal::tree_args(ctx, pool, slots, q_start, n_seqs, rows);
    a.q = q;
    a.out = out;
    a.k = static_cast<const char*>(pool->stores[k_store]);
    a.v = static_cast<const char*>(pool->stores[v_store]);
    a.mask = reinterpret_cast<const unsigned long long*>(mask);
    a.mask_words = mask_words;
    a.q_stride = q_row_stride;
    a.out_stride = out_row_stride;
    a.n_q_heads = n_q_heads;
    a.n_kv_heads = n_kv_heads;
    a.group = n_q_heads / n_kv_heads;
    a.head_dim = head_dim;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.wait_limit = static_cast<unsigned>(lokal::tune_env("LOKAL_CUDA_WAIT_LIMIT", lokal::kWaitLimit));
    a.extra_tx = static_cast<unsigned>(lokal::tune_env("LOKAL_CUDA_TEST_EXTRA_TX", 0));
    cudaStream_t st = static_cast<cudaStream_t>(s);
    a.out_vec32 = lokal::aligned_to(out, 32) && out_row_stride * es % 32 == 0;
    const bool tc = lokal::tree_tc_takes(a, dtype, kv_dtype), mma = !tc && lokal::tree_mma_takes(a, dtype, kv_dtype);
    a.block_rows = tc ? lokal::tree_tc_block(a) : 16u;
    a.part_ml = static_cast<float2*>(workspace);
    a.part_o = reinterpret_cast<float*>(a.part_ml + (tc ? lokal::tree_tc_rows(ctx) : mma ? lokal::tree_mma_rows(ctx, head_dim) : lokal::any_rows(ctx, head_dim)));
    if (tc) return lokal::launch_tree_tc(ctx, st, a, dtype);
    if (mma) return lokal::launch_tree_mma(ctx, st, a, dtype, kv_dtype);
    switch (dtype) {
        case LOKAL_F32: return lokal::launch_any_q<float>(ctx, st, a, kv_dtype);
        case LOKAL_F16: return lokal::launch_any_q<__half>(ctx, st, a, kv_dtype);
        default: return lokal::launch_any_q<__nv_bfloat16>(ctx, st, a, kv_dtype);
    }
}

}  // extern "C"
