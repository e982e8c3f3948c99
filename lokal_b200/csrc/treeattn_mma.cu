// Attention of drafted rows over a paged cache with f32 accuracy on the tensor cores: f32 query rows over a cache of any
// type, 16-bit ones over a cache of another type; head sizes 64 and 128.
//
// tf32 products take 11 significant bits of each factor. A value of f16 or bf16 has no more; an f32 value is split into
// two parts, x = hi + lo with hi x rounded to 11 bits and lo the rest rounded to 11, and a product into hi*hi + hi*lo + lo*hi (what is
// left out is below 2^-22 of it; a factor that needs no split drops its term). So the weights, which stay f32, and the
// query rows cost two products a piece over a 16-bit cache and three over an f32 one. Sums over the keys are taken per
// step of 8 or 16 keys in the tensor core and joined in f32 on the outside.
//
// An infinity does not survive the split (inf - inf is NaN, and an infinity times the parts of a factor has either sign), nor
// do the largest f32 values, which round up to one. Wherever that happens to what a row sees, the row's sums are not finite. So
// a warp that ends a block with such sums goes through its keys again, with care: scores that are not finite are summed as
// plain f32 products, and such values of V are left out of the product and added one by one. (With care from the first, always:
// 16 sequences of 20,000 keys, 4 rows each, 16 / 8 heads of 128, f32 over f16 took 554 us, and 472 so.)
//
// Bound by memory at few rows (a step of 16 keys of 128 columns is 8 KB of f16 cache and 128 products of 16 x 8 x 8).
// Every warp is on its own: it walks every fourth run of keys of the CTA's tiles, fetches K and V from the pages straight
// into the registers in which the product wants them, and the next K while it weighs this one; eight warps to an SM keep
// 64 KB on their way. The order of the contraction is free, so the fragments are cut such that a thread's share of a row
// is 32 contiguous bytes. The four warps' sums are put together when the block ends.
#include "treeattn.cuh"

namespace lokal {
namespace {

constexpr int kMmaRows = 16, kMmaKeys = 64, kMmaThreads = 128;

template <typename T>
struct Split {  // whether a value of the type needs a second tf32 part
    static constexpr bool value = sizeof(T) == 4;
};

// Both parts are rounded, not cut off: half a step of 2^-12 each instead of a whole one that always points to zero.
__device__ __forceinline__ uint32_t tf32_round(float x) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t tf32_hi(float x) { return tf32_round(x); }
__device__ __forceinline__ uint32_t tf32_lo(float x, uint32_t hi) { return tf32_round(x - __uint_as_float(hi)); }

// Whether a value of type T goes into the product: finite, and so when it is rounded to 11 bits.
constexpr float kTf32Over = 1.0009765625f;  // 1 + 2^-10: at least a step of tf32
template <typename T>
__device__ __forceinline__ bool tf32_holds(float x) { return isfinite(Split<T>::value ? x * kTf32Over : x); }
// The same of a whole word of a run, many of them in a sum: adds 0 to t, or NaN if a value does not go into the product.
template <typename T>
__device__ __forceinline__ uint32_t run_word(uint32_t w, uint32_t t);
template <>
__device__ __forceinline__ uint32_t run_word<float>(uint32_t w, uint32_t t) { return __float_as_uint(fmaf(__uint_as_float(w) * kTf32Over, 0.0f, __uint_as_float(t))); }
template <>
__device__ __forceinline__ uint32_t run_word<__half>(uint32_t w, uint32_t t) {
    const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&w), __floats2half2_rn(0.0f, 0.0f), *reinterpret_cast<const __half2*>(&t));
    return *reinterpret_cast<const uint32_t*>(&r);
}
template <>
__device__ __forceinline__ uint32_t run_word<__nv_bfloat16>(uint32_t w, uint32_t t) {
    const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w), __floats2bfloat162_rn(0.0f, 0.0f), *reinterpret_cast<const __nv_bfloat162*>(&t));
    return *reinterpret_cast<const uint32_t*>(&r);
}
// whether t, a sum of zeros of either sign, has become NaN (in either half)
template <typename T>
__device__ __forceinline__ bool run_odd(uint32_t t) { return (t & (Split<T>::value ? 0x7fffffffu : 0x7fff7fffu)) != 0u; }

// c += a b over a contraction of 8: a 16 x 8, b 8 x 8
__device__ __forceinline__ void mma_tf32(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 32 contiguous bytes (16 and zeros, with HALF)
struct Run32 {
    uint32_t w[8];
};
template <bool HALF>
__device__ __forceinline__ Run32 load_run(const void* p) {
    Run32 r;
    if (HALF) {
        const uint4 v = ld_stream(p);
        r.w[0] = v.x, r.w[1] = v.y, r.w[2] = v.z, r.w[3] = v.w;
        r.w[4] = r.w[5] = r.w[6] = r.w[7] = 0u;
    } else
        asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]), "=r"(r.w[7])
                     : "l"(p));
    return r;
}
// element e of a run
template <typename T>
__device__ __forceinline__ float elem(const Run32& r, int e);
template <>
__device__ __forceinline__ float elem<float>(const Run32& r, int e) { return __uint_as_float(r.w[e]); }
template <>
__device__ __forceinline__ float elem<__nv_bfloat16>(const Run32& r, int e) { return __uint_as_float(e & 1 ? r.w[e / 2] & 0xffff0000u : r.w[e / 2] << 16); }
template <>
__device__ __forceinline__ float elem<__half>(const Run32& r, int e) {
    const __half2 h = *reinterpret_cast<const __half2*>(&r.w[e / 2]);
    return e & 1 ? __high2float(h) : __low2float(h);
}

template <int HD>
struct MmaShape {
    static constexpr size_t kQ = HD / 8 * 32 * 8 * 4;                   // query fragments, hi and lo
    static constexpr size_t kO = 4 * kMmaRows * (HD + 4) * 4;           // the warps' sums (rows padded off the banks)
    static constexpr size_t kBytes = (kQ > kO ? kQ : kO) + 4 * kMmaRows * 8 + 16 * 8;
};

template <typename TQ, typename TK, int HD>
__global__ void __launch_bounds__(kMmaThreads, HD == 64 ? 4 : 2) tree_attn_mma_kernel(const __grid_constant__ TreeArgs a) {
    pdl_sync();
    constexpr int E = 32 / sizeof(TK);         // elements of a 32-byte run
    constexpr int SUP = HD / (4 * E);          // runs of a K row to a thread
    constexpr int NT = sizeof(TK) == 4 ? 1 : 2;  // groups of 8 keys to a step
    constexpr int VR = (HD / 8 + E - 1) / E;   // runs of a V row to a thread (with 64 columns of 16 bits, half a run)
    constexpr bool SQ = Split<TQ>::value, SK = Split<TK>::value;
    extern __shared__ __align__(16) unsigned char smem[];
    uint4* qf = reinterpret_cast<uint4*>(smem);  // [HD / 8 steps][32 lanes][hi, lo]
    float* osum = reinterpret_cast<float*>(smem);
    float2* ml = reinterpret_cast<float2*>(smem + (MmaShape<HD>::kQ > MmaShape<HD>::kO ? MmaShape<HD>::kQ : MmaShape<HD>::kO));
    unsigned long long* sh = reinterpret_cast<unsigned long long*>(ml + 4 * kMmaRows);
    const unsigned tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, g = lane >> 2, c = lane & 3u;
    const unsigned shares = gridDim.x;
    const TreePlace place = tree_locate<kMmaKeys, kMmaThreads>(a, sh, blockIdx.x == 0, [&](unsigned total) {
        const TreeShares s(total, shares);
        return blockIdx.x < s.g ? s.first(blockIdx.x) : total;
    });
    if (place.seq >= a.n_seqs) return;
    const TreeShares share(place.total, shares);
    TreeWalk<kMmaKeys> walk;
    walk.start(a, place, share.first(blockIdx.x), share.first(blockIdx.x + 1));
    TreeUnit u;
    while (walk.next(a, u)) {
        const unsigned rows_all = u.seq.n * a.group, flat0 = u.block * kMmaRows, m_rows = min(static_cast<unsigned>(kMmaRows), rows_all - flat0);
        // The block's rows as fragments: at step s of run p, thread (g, c) takes columns 4E p + E c + 2 s and the next one of
        // rows g and g + 8, the columns that its K run holds.
        __syncthreads();
        for (unsigned e = tid; e < HD / 8 * 32; e += kMmaThreads) {
            const unsigned step = e / 32, ln = e % 32, col = step / (E / 2) * 4 * E + (ln & 3u) * E + step % (E / 2) * 2;
            float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // (row g, first), (row g + 8, first), (row g, second), (row g + 8, second)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const unsigned r = (ln >> 2) + 8 * h;
                if (r < m_rows) {
                    const unsigned flat = flat0 + r, node = flat / a.group, head = u.kv_head * a.group + flat % a.group;
                    const TQ* q = static_cast<const TQ*>(a.q) + static_cast<size_t>(u.seq.row0 + node) * a.q_stride + static_cast<size_t>(head) * HD + col;
                    x[h] = to_f32<TQ>(q[0]);
                    x[2 + h] = to_f32<TQ>(q[1]);
                }
            }
            const uint4 hi = make_uint4(tf32_hi(x[0]), tf32_hi(x[1]), tf32_hi(x[2]), tf32_hi(x[3]));
            qf[2 * e] = hi;
            qf[2 * e + 1] = make_uint4(tf32_lo(x[0], hi.x), tf32_lo(x[1], hi.y), tf32_lo(x[2], hi.z), tf32_lo(x[3], hi.w));
        }
        __syncthreads();
        const unsigned node0 = (flat0 + min(g, m_rows - 1)) / a.group, node1 = (flat0 + min(g + 8, m_rows - 1)) / a.group;
        float o[HD / 8][4];
#pragma unroll
        for (int j = 0; j < HD / 8; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};  // rows g and g + 8
        const char* k_base = a.k + (static_cast<size_t>(u.kv_head) * HD + c * E) * sizeof(TK);
        const char* v_base = a.v + (static_cast<size_t>(u.kv_head) * HD + g * (HD / 8)) * sizeof(TK);
        // the warp's steps: 8 * NT keys each, 64 / (8 * NT) of them to a tile, dealt to the four warps in turn
        constexpr unsigned kStep = 8 * NT;
        const unsigned pos_end = min(u.k1 * kMmaKeys, static_cast<unsigned>(u.seq.len));
        const auto row_at = [&](unsigned pos) -> unsigned {  // cache row of key pos + (lane % kStep)
            const unsigned p = pos + lane % kStep;
            if (p >= pos_end) return 0u;
            return (tree_page(a, u.seq.slot, p >> a.page_shift) << a.page_shift) + (p & (a.page_rows - 1));
        };
        unsigned pos = u.k0 * kMmaKeys + warp * kStep;
        unsigned rows_now = row_at(pos), rows_next = row_at(pos + 4 * kStep);
        Run32 kr[NT][SUP];
        // (Keys behind the last one are read from row 0, without a branch: nobody sees them, and their V is cleared.)
        const auto load_k = [&](unsigned rows) {
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const unsigned row = __shfl_sync(0xffffffffu, rows, n * 8 + g);
                const char* at = k_base + row * a.row_bytes;
#pragma unroll
                for (int s = 0; s < SUP; s++) kr[n][s] = load_run<false>(at + s * 4 * 32);
            }
        };
        if (pos < pos_end) load_k(rows_now);
        bool careful = false;
        for (;; pos += 4 * kStep) {
            if (pos >= pos_end) {
                if (careful) break;
                float zero = l[0] * 0.0f + l[1] * 0.0f;
#pragma unroll
                for (int j = 0; j < HD / 8; j++) zero += (o[j][0] * 0.0f + o[j][1] * 0.0f) + (o[j][2] * 0.0f + o[j][3] * 0.0f);
                if (__all_sync(0xffffffffu, zero == 0.0f)) break;
                careful = true;
#pragma unroll
                for (int j = 0; j < HD / 8; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
                m[0] = m[1] = -INFINITY;
                l[0] = l[1] = 0.0f;
                pos = u.k0 * kMmaKeys + warp * kStep;
                rows_now = row_at(pos);
                rows_next = row_at(pos + 4 * kStep);
                load_k(rows_now);
            }
            // V of the step: keys 2c and 2c + 1 of each group of 8, columns (HD / 8) g and on
            Run32 vr[NT][2][VR];
#pragma unroll
            for (int n = 0; n < NT; n++) {
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const unsigned row = __shfl_sync(0xffffffffu, rows_now, n * 8 + 2 * c + h);
                    const char* at = v_base + row * a.row_bytes;
#pragma unroll
                    for (int r = 0; r < VR; r++) vr[n][h][r] = load_run<(HD / 8 < E)>(at + r * 32);
                }
            }
            // In several sums, put together in f32: a tensor core cuts a sum off where f32 would round it, and one long chain
            // of products shows it (f32 over f32 with 128 columns: 1.2e-6 of the result, 0.33e-6 so).
            constexpr int CH = NT == 1 ? 4 : 2;
            float zs[CH][NT][4];
#pragma unroll
            for (int n = 0; n < NT * CH; n++) zs[n / NT][n % NT][0] = zs[n / NT][n % NT][1] = zs[n / NT][n % NT][2] = zs[n / NT][n % NT][3] = 0.0f;
#pragma unroll
            for (int s = 0; s < SUP; s++) {
#pragma unroll
                for (int t = 0; t < E / 2; t++) {
                    const uint4 hi = qf[((s * (E / 2) + t) * 32 + lane) * 2];
                    uint4 lo = make_uint4(0u, 0u, 0u, 0u);
                    if (SQ) lo = qf[((s * (E / 2) + t) * 32 + lane) * 2 + 1];
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        const float k0 = elem<TK>(kr[n][s], 2 * t), k1 = elem<TK>(kr[n][s], 2 * t + 1);
                        const uint32_t h0 = SK ? tf32_hi(k0) : __float_as_uint(k0), h1 = SK ? tf32_hi(k1) : __float_as_uint(k1);
                        float(&zc)[4] = zs[(s * (E / 2) + t) % CH][n];
                        if (SQ) mma_tf32(zc, lo.x, lo.y, lo.z, lo.w, h0, h1);
                        if (SK) mma_tf32(zc, hi.x, hi.y, hi.z, hi.w, tf32_lo(k0, h0), tf32_lo(k1, h1));
                        mma_tf32(zc, hi.x, hi.y, hi.z, hi.w, h0, h1);
                    }
                }
            }
            float z[NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++) {
#pragma unroll
                for (int i = 0; i < 4; i++) z[n][i] = CH == 4 ? (zs[0][n][i] + zs[1][n][i]) + (zs[2 % CH][n][i] + zs[3 % CH][n][i]) : zs[0][n][i] + zs[1][n][i];
            }
            if ((SQ || SK) && careful) {
#pragma unroll
                for (int n = 0; n < NT; n++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const unsigned row = __shfl_sync(0xffffffffu, rows_now, n * 8 + 2 * c + (i & 1));
                        if (isfinite(z[n][i])) continue;
                        const unsigned flat = flat0 + min(g + 8 * (i >> 1), m_rows - 1), node = flat / a.group, head = u.kv_head * a.group + flat % a.group;
                        const TQ* q = static_cast<const TQ*>(a.q) + static_cast<size_t>(u.seq.row0 + node) * a.q_stride + static_cast<size_t>(head) * HD;
                        const TK* k = reinterpret_cast<const TK*>(a.k + row * a.row_bytes) + static_cast<size_t>(u.kv_head) * HD;
                        float sum = 0.0f;
#pragma unroll 1
                        for (int d = 0; d < HD; d++) sum = fmaf(to_f32<TQ>(q[d]), to_f32<TK>(k[d]), sum);
                        z[n][i] = sum;
                    }
                }
            }
            const unsigned next = pos + 4 * kStep;
            if (next < pos_end) {
                load_k(rows_next);
                rows_now = rows_next;
                rows_next = row_at(next + 4 * kStep);
            }
            // weights
            const bool masked = static_cast<int>(pos + kStep) > u.seq.ctx;
            unsigned seen[2] = {0xffffffffu, 0xffffffffu};
            if (masked) {
                seen[0] = tree_visible(a, u.seq, node0, static_cast<int>(pos)) >> (2 * c);
                seen[1] = tree_visible(a, u.seq, node1, static_cast<int>(pos)) >> (2 * c);
                if (pos + kStep > pos_end) {  // keys of the next share
                    const unsigned in = ((1u << (pos_end - pos)) - 1u) >> (2 * c);
                    seen[0] &= in;
                    seen[1] &= in;
                }
            }
            float scale[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float top = -INFINITY;
#pragma unroll
                for (int n = 0; n < NT; n++) {
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float& x = z[n][2 * h + e];
                        x = (seen[h] >> (8 * n + e)) & 1u ? x * a.scale_log2 : -INFINITY;
                        top = fmaxf(top, x);
                    }
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                top = fmaxf(top, m[h]);
                const float ref = top == -INFINITY ? 0.0f : top;
                scale[h] = exp2f(m[h] - ref);
                m[h] = top;
                float sum = 0.0f;
#pragma unroll
                for (int n = 0; n < NT; n++) {
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float& x = z[n][2 * h + e];
                        x = (seen[h] >> (8 * n + e)) & 1u ? exp2f(x - ref) : 0.0f;
                        sum += x;
                    }
                }
                l[h] = fmaf(l[h], scale[h], sum);  // of this thread's keys; the four threads of a row are added at the end
            }
            // Values of V that do not go into the product are taken out of it and added one by one; where there are drafted rows,
            // the first time through as well: they would reach the rows that do not see them, as 0 times an infinity.
            if (pos + kStep > pos_end) {
#pragma unroll
                for (int n = 0; n < NT; n++) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        if (pos + n * 8 + 2 * c + h < pos_end) continue;
#pragma unroll
                        for (int r = 0; r < VR; r++) {
#pragma unroll
                            for (int e = 0; e < 8; e++) vr[n][h][r].w[e] = 0u;
                        }
                    }
                }
            }
            bool bad = false;
            if (masked || careful) {
                uint32_t zeros[2] = {0u, 0u};
#pragma unroll
                for (int n = 0; n < NT; n++) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
#pragma unroll
                        for (int r = 0; r < VR; r++) {
#pragma unroll
                            for (int e = 0; e < (HD / 8 < E ? 4 : 8); e++) zeros[h] = run_word<TK>(vr[n][h][r].w[e], zeros[h]);
                        }
                    }
                }
                bad = __any_sync(0xffffffffu, run_odd<TK>(zeros[0]) || run_odd<TK>(zeros[1]));
            }
            if (bad) {
#pragma unroll
                for (int n = 0; n < NT; n++) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
#pragma unroll
                        for (int r = 0; r < VR; r++) {
#pragma unroll
                            for (int e = 0; e < 8; e++)
                                if (sizeof(TK) == 4) {
                                    if (!tf32_holds<TK>(elem<TK>(vr[n][h][r], e))) vr[n][h][r].w[e] = 0u;
                                } else {
                                    if (!tf32_holds<TK>(elem<TK>(vr[n][h][r], (2 * e) % E))) vr[n][h][r].w[e] &= 0xffff0000u;
                                    if (!tf32_holds<TK>(elem<TK>(vr[n][h][r], (2 * e + 1) % E))) vr[n][h][r].w[e] &= 0x0000ffffu;
                                }
                        }
                    }
                }
            }
            // O = O * scale + P V: column 2c + e of product j is column (HD / 8) (2c + e) + j of the row
            uint32_t p_hi[NT][4], p_lo[NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    p_hi[n][i] = tf32_hi(z[n][i]);
                    p_lo[n][i] = tf32_lo(z[n][i], p_hi[n][i]);
                }
            }
#pragma unroll
            for (int j = 0; j < HD / 8; j++) {
                float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    const float v0 = elem<TK>(vr[n][0][j / E], j % E), v1 = elem<TK>(vr[n][1][j / E], j % E);
                    const uint32_t h0 = SK ? tf32_hi(v0) : __float_as_uint(v0), h1 = SK ? tf32_hi(v1) : __float_as_uint(v1);
                    mma_tf32(x, p_lo[n][0], p_lo[n][2], p_lo[n][1], p_lo[n][3], h0, h1);
                    if (SK) mma_tf32(x, p_hi[n][0], p_hi[n][2], p_hi[n][1], p_hi[n][3], tf32_lo(v0, h0), tf32_lo(v1, h1));
                    mma_tf32(x, p_hi[n][0], p_hi[n][2], p_hi[n][1], p_hi[n][3], h0, h1);
                }
#pragma unroll
                for (int i = 0; i < 4; i++) o[j][i] = fmaf(o[j][i], scale[i >> 1], x[i]);
            }
            if (bad) {
                for (unsigned key = 0; key < kStep; key++) {
                    const unsigned from = (lane & ~3u) + (key % 8) / 2;  // the thread of this row that has the key's weight
                    float w[2];
                    unsigned sees[2];
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        float mine = 0.0f;
#pragma unroll
                        for (int n = 0; n < NT; n++) {
#pragma unroll
                            for (int e = 0; e < 2; e++)
                                if (key / 8 == static_cast<unsigned>(n) && key % 2 == static_cast<unsigned>(e)) mine = z[n][2 * h + e];
                        }
                        w[h] = __shfl_sync(0xffffffffu, mine, from);
                        sees[h] = __shfl_sync(0xffffffffu, (seen[h] >> (8 * (key / 8) + key % 2)) & 1u, from);
                    }
                    const unsigned p = pos + key;
                    if (p >= pos_end) continue;
                    const size_t row = (static_cast<size_t>(tree_page(a, u.seq.slot, p >> a.page_shift)) << a.page_shift) + (p & (a.page_rows - 1));
                    const TK* v = reinterpret_cast<const TK*>(a.v + row * a.row_bytes) + static_cast<size_t>(u.kv_head) * HD;
#pragma unroll
                    for (int j = 0; j < HD / 8; j++) {
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const float x = to_f32<TK>(v[(HD / 8) * (2 * c + e) + j]);
                            if (tf32_holds<TK>(x)) continue;
                            if (sees[0]) o[j][e] += w[0] * x;
                            if (sees[1]) o[j][2 + e] += w[1] * x;
                        }
                    }
                }
            }
        }
        // the four warps together
        __syncthreads();  // the query fragments make way for the sums
#pragma unroll
        for (int h = 0; h < 2; h++) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            if (c == 0) ml[warp * kMmaRows + g + 8 * h] = make_float2(m[h], l[h]);
        }
#pragma unroll
        for (int j = 0; j < HD / 8; j++) {
#pragma unroll
            for (int i = 0; i < 4; i++) osum[(warp * kMmaRows + g + 8 * (i >> 1)) * (HD + 4) + (HD / 8) * (2 * c + (i & 1)) + j] = o[j][i];
        }
        __syncthreads();
        for (unsigned e = tid; e < kMmaRows * HD; e += kMmaThreads) {
            const unsigned r = e / HD, col = e % HD;
            if (r >= m_rows) break;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < 4; w++) top = fmaxf(top, ml[w * kMmaRows + r].x);
            const float ref = top == -INFINITY ? 0.0f : top;
            float sum = 0.0f, x = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float2 t = ml[w * kMmaRows + r];
                const float f = t.y == 0.0f ? 0.0f : exp2f(t.x - ref);
                sum = fmaf(t.y, f, sum);
                x = f == 0.0f ? x : fmaf(osum[(w * kMmaRows + r) * (HD + 4) + col], f, x);
            }
            if (u.whole) {
                const unsigned flat = flat0 + r, node = flat / a.group, head = u.kv_head * a.group + flat % a.group;
                static_cast<TQ*>(a.out)[static_cast<size_t>(u.seq.row0 + node) * a.out_stride + static_cast<size_t>(head) * HD + col] =
                    from_f32<TQ>(sum == 0.0f ? 0.0f : x / sum);
            } else {
                const size_t piece = (static_cast<size_t>(blockIdx.x) * 2 + u.piece) * kMmaRows + r;
                a.part_o[piece * HD + col] = x;
                if (col == 0) a.part_ml[piece] = make_float2(top, sum);
            }
        }
    }
}

constexpr unsigned mma_ctas(unsigned head_dim) { return head_dim == 64 ? 4 : 2; }  // to an SM: what the registers allow

template <typename TQ, typename TK, int HD>
int launch_mma(lokal_cuda_ctx* ctx, cudaStream_t s, const TreeArgs& a) {
    const unsigned shares = static_cast<unsigned>(ctx->sm_count) * mma_ctas(HD);
    launch_staged(tree_attn_mma_kernel<TQ, TK, HD>, shares, kMmaThreads, MmaShape<HD>::kBytes, s, a);
    LOKAL_CHECK_LAUNCH(ctx, "tree_attn_mma_kernel");
    launch_k(tree_join_kernel<TQ, kMmaRows, kMmaKeys>, shares - 1, 256, 0, s, a, shares);
    LOKAL_CHECK_LAUNCH(ctx, "tree_join_kernel");
    return LOKAL_OK;
}

template <typename TQ, typename TK>
int launch_mma_hd(lokal_cuda_ctx* ctx, cudaStream_t s, const TreeArgs& a) {
    return a.head_dim == 64 ? launch_mma<TQ, TK, 64>(ctx, s, a) : launch_mma<TQ, TK, 128>(ctx, s, a);
}

}  // namespace

size_t tree_mma_rows(const lokal_cuda_ctx* ctx, unsigned head_dim) { return static_cast<size_t>(ctx->sm_count) * mma_ctas(head_dim) * 2 * kMmaRows; }

bool tree_mma_takes(const TreeArgs& a, int dtype, int kv_dtype) {
    return (a.head_dim == 64 || a.head_dim == 128) && (dtype == LOKAL_F32 || dtype != kv_dtype) && a.row_bytes % 32 == 0 && aligned_to(a.k, 32) && aligned_to(a.v, 32);
}

int launch_tree_mma(lokal_cuda_ctx* ctx, cudaStream_t s, const TreeArgs& a, int dtype, int kv_dtype) {
    if (dtype == LOKAL_F32) {
        if (kv_dtype == LOKAL_F32) return launch_mma_hd<float, float>(ctx, s, a);
        if (kv_dtype == LOKAL_F16) return launch_mma_hd<float, __half>(ctx, s, a);
        return launch_mma_hd<float, __nv_bfloat16>(ctx, s, a);
    }
    if (dtype == LOKAL_F16) return kv_dtype == LOKAL_F32 ? launch_mma_hd<__half, float>(ctx, s, a) : launch_mma_hd<__half, __nv_bfloat16>(ctx, s, a);
    return kv_dtype == LOKAL_F32 ? launch_mma_hd<__nv_bfloat16, float>(ctx, s, a) : launch_mma_hd<__nv_bfloat16, __half>(ctx, s, a);
}

}  // namespace lokal
