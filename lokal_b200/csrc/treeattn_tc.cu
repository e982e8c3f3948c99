// Attention of drafted rows over a paged cache on the tensor cores: 16-bit rows of the cache's own type, head sizes 64
// and 128. The other types and shapes run in treeattn.cu; the mathematics and the walk over the work are in treeattn.cuh.
//
// Bound by memory up to about 250 query rows per key head (a key and its value are 4 * head_dim bytes and cost
// 4 * head_dim flops per row; the measured 1634 TFLOP/s over 6570 GB/s are 249 flops per byte), so the aim is that the
// copies never wait. One CTA per SM, 128 query rows by 128 keys:
//   warp 8      brings K and V tiles, page by page, into a ring of stages with TMA (128-byte swizzle)
//   warp 9      issues the products: S = Q K^T into TMEM, O += P V with P read from TMEM and V as it lies (MN-major)
//   warps 0-3   take the even tiles, warps 4-7 the odd ones: S from TMEM, maximum, exp2, P back over S
// The two groups of warps are two streams of the running softmax, each with a maximum, a sum and an accumulator of its
// own, so neither waits for the other, and the product of one tile runs while the other group works on its own; they
// are put together when the block ends. An accumulator is rescaled only when the maximum has grown by more than 2^8
// since it was last set: weights then stay below 2^8, which neither 16-bit type nor the f32 sums mind.
// Weights are rounded to the cache's type for the product (half a step each, as the values they multiply were); sums,
// maxima and scores are f32.
#include <cuda.h>

#include "treeattn.cuh"

namespace lokal {
namespace {

constexpr int kTcRows = 128, kTcKeys = 128, kTcThreads = 320;
constexpr int kSoftmaxThreads = 256;

template <int HD>
struct TcShape {
    static constexpr int kSubs = HD / 64;                   // 64-column panels of 128 bytes
    static constexpr unsigned kPanel = 128 * 128;           // bytes of a panel of 128 rows
    static constexpr unsigned kTile = kSubs * kPanel;       // bytes of a K or V tile, and of Q
    static constexpr int kStages = HD == 128 ? 3 : 6;       // 192 KB either way
    static constexpr unsigned kMl = kTile + kStages * 2 * kTile;        // float2[2][128]
    static constexpr unsigned kBars = kMl + 2 * 128 * 8;                // mbarriers
    static constexpr unsigned kNumBars = (3 * kStages + 6 + 1) / 2 * 2;
    static constexpr unsigned kMisc = kBars + kNumBars * 8;             // TMEM address, flags
    static constexpr unsigned kBytes = kMisc + 32;
    static_assert(kBytes <= 227 * 1024, "a CTA's shared memory");
};

// ---- tcgen05 ----
__device__ __forceinline__ void tc_alloc(uint32_t dst, unsigned cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(cols) : "memory");
}
__device__ __forceinline__ void tc_dealloc(uint32_t tmem, unsigned cols) {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols));
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t mbar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(mbar) : "memory");
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// D[tmem] (+)= A[smem] B[smem]
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(static_cast<unsigned>(add))
        : "memory");
}
// D[tmem] (+)= A[tmem] B[smem]
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(static_cast<unsigned>(add))
        : "memory");
}

#define TC_R4(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3])
#define TC_W4(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3])
// 32 columns of the warp's 32 lanes; one lane per thread
__device__ __forceinline__ void tc_ld32(uint32_t at, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
        "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : TC_R4(v, 0), TC_R4(v, 4), TC_R4(v, 8), TC_R4(v, 12), TC_R4(v, 16), TC_R4(v, 20), TC_R4(v, 24), TC_R4(v, 28)
        : "r"(at));
}
__device__ __forceinline__ void tc_st32(uint32_t at, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,"
        "%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at),
        TC_W4(v, 0), TC_W4(v, 4), TC_W4(v, 8), TC_W4(v, 12), TC_W4(v, 16), TC_W4(v, 20), TC_W4(v, 24), TC_W4(v, 28)
        : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t at, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at), TC_W4(v, 0),
        TC_W4(v, 4), TC_W4(v, 8), TC_W4(v, 12)
        : "memory");
}

// Shared-memory operand with the 128-byte swizzle. K-major (Q, K): rows of 128 bytes, groups of 8 rows 1024 bytes apart.
// MN-major (V: the output columns are contiguous, the keys are rows): 64-column panels `kPanel` apart, groups of 8 keys
// 1024 bytes apart.
__device__ __forceinline__ uint64_t tc_desc(uint32_t addr, unsigned leading) {
    return static_cast<uint64_t>((addr & 0x3ffffu) >> 4) | (static_cast<uint64_t>(leading >> 4) << 16) | (static_cast<uint64_t>(1024u >> 4) << 32) |
           (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}
// f32 accumulator, both operands f16 (0) or bf16 (1), 128 rows by n columns; b_mn: B is MN-major
__device__ __forceinline__ constexpr uint32_t tc_idesc(unsigned fmt, unsigned n, unsigned b_mn) {
    return (1u << 4) | (fmt << 7) | (fmt << 10) | (b_mn << 16) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

__device__ __forceinline__ void mbar_arrive(uint32_t mbar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(mbar) : "memory"); }
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t mbar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(mbar)
                 : "memory");
}
__device__ __forceinline__ void bar_softmax() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {  // 2 steps of error, 0 for results below the smallest normal value
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// whether one of the two values is an infinity or a NaN
template <typename T>
__device__ __forceinline__ bool bad_pair(uint32_t v) {
    constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    return (v & e) == e || ((v >> 16) & e) == e;
}

// A wait that gives up: after `limit` polls, or when another role of the CTA has.
__device__ __forceinline__ bool tc_wait(uint32_t mbar, unsigned parity, unsigned limit, volatile int* gave_up) {
    if (mbar_try_wait(mbar, parity)) return true;
    for (unsigned spin = 0; spin < limit; spin++) {
        if (mbar_try_wait(mbar, parity)) return true;
        if ((spin & 63u) == 63u && *gave_up) return false;
    }
    *gave_up = 1;
    return false;
}

// V rows that hold an infinity or a NaN and belong to drafted rows were cleared for the product, because rows that do not
// see them would get 0 * inf. What they add to the rows that do see them is added here, to the stored result: rare, and
// slow (a dot product per row and value).
template <typename T, int HD>
__device__ __noinline__ void add_bad_values(const TreeArgs& a, const TreeUnit& u, unsigned node, unsigned head, float m, float l, T* out, float* piece,
                                            unsigned c0, unsigned c1) {
    const int first = max(u.seq.ctx, static_cast<int>(u.k0) * kTcKeys), last = min(u.seq.len, static_cast<int>(u.k1) * kTcKeys);
    const T* q = static_cast<const T*>(a.q) + static_cast<size_t>(u.seq.row0 + node) * a.q_stride + static_cast<size_t>(head) * HD;
    for (int pos = first; pos < last; pos++) {
        if (!(tree_visible(a, u.seq, node, pos) & 1u)) continue;
        const size_t row = (static_cast<size_t>(tree_page(a, u.seq.slot, static_cast<unsigned>(pos) >> a.page_shift)) << a.page_shift) +
                           (static_cast<unsigned>(pos) & (a.page_rows - 1));
        const size_t off = row * a.row_bytes + static_cast<size_t>(u.kv_head) * HD * 2;
        const T* v = reinterpret_cast<const T*>(a.v + off);
        const T* k = reinterpret_cast<const T*>(a.k + off);
        float p = 0.0f;
        bool have = false;
        for (unsigned c = c0; c < c1; c++) {
            const float x = to_f32<T>(v[c]);
            if (isfinite(x)) continue;
            if (!have) {
                float s = 0.0f;
                for (int d = 0; d < HD; d++) s = fmaf(to_f32<T>(q[d]), to_f32<T>(k[d]), s);
                p = exp2f(fmaf(s, a.scale_log2, -m));
                have = true;
            }
            if (piece) piece[c] += p * x;
            else out[c] = from_f32<T>(to_f32<T>(out[c]) + p * x / l);
        }
    }
}

template <typename T, int HD>
__global__ void __launch_bounds__(kTcThreads, 1)
    tree_attn_tc_kernel(const TreeArgs a, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
    using S = TcShape<HD>;
    extern __shared__ __align__(1024) unsigned char tc_smem[];
    const uint32_t smem = smem_addr(tc_smem);
    const unsigned tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const uint32_t bars = smem + S::kBars;
    auto kfull = [&](int st) { return bars + st * 8; };
    auto vfull = [&](int st) { return bars + (S::kStages + st) * 8; };
    auto empty = [&](int st) { return bars + (2 * S::kStages + st) * 8; };
    const uint32_t sfull = bars + 3 * S::kStages * 8, pready = sfull + 16, qfull = sfull + 32, udone = sfull + 40;
    volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(tc_smem + S::kMisc);  // [0] TMEM, [1] a wait gave up, [2], [3] bad values in a unit
    volatile int* gave_up = reinterpret_cast<volatile int*>(misc + 1);
    float2* ml = reinterpret_cast<float2*>(tc_smem + S::kMl);
    // set-up that touches no global memory goes ahead of the wait for the launch before
    if (warp == 8) {
        tc_alloc(smem + S::kMisc, 512);
        if (lane == 0) {
            for (int st = 0; st < S::kStages; st++) {
                mbar_init(kfull(st), 1);
                mbar_init(vfull(st), 1);
                mbar_init(empty(st), 1);
            }
            for (int w = 0; w < 2; w++) {
                mbar_init(sfull + 8 * w, 1);
                mbar_init(pready + 8 * w, 128);
            }
            mbar_init(qfull, kSoftmaxThreads);
            mbar_init(udone, 1);
            mbar_init_fence();
            misc[1] = misc[2] = misc[3] = 0;
        }
    }
    pdl_sync();
    // the ring is not in use yet: it holds the sums of the walk
    const unsigned shares = gridDim.x;
    const TreePlace place = tree_locate<kTcRows, kTcKeys, kTcThreads>(a, reinterpret_cast<unsigned long long*>(tc_smem), blockIdx.x == 0, [&](unsigned long long total) {
        const unsigned g = total < shares ? static_cast<unsigned>(total) : shares;
        return blockIdx.x < g ? tree_share(total, blockIdx.x, g) : total;
    });
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = misc[0];
    const unsigned g = place.total < shares ? static_cast<unsigned>(place.total) : shares;
    TreeWalk<kTcRows, kTcKeys> walk;
    walk.start(a, place, place.seq < a.n_seqs ? tree_share(place.total, blockIdx.x, g) : 0, place.seq < a.n_seqs ? tree_share(place.total, blockIdx.x + 1, g) : 0);
    TreeUnit u;
    bool ok = place.seq < a.n_seqs;

    if (warp == 8) {
        // ---- K and V tiles ----
        unsigned t = 0;  // tiles so far
        const unsigned box_rows = min(a.page_rows, static_cast<unsigned>(kTcKeys));
        while (ok && walk.next(a, u)) {
            for (unsigned kt = u.k0; ok && kt < u.k1; kt++, t++) {
                const int st = static_cast<int>(t % S::kStages);
                const unsigned round = t / S::kStages;
                if (round) ok = tc_wait(empty(st), (round - 1) & 1u, a.wait_limit, gave_up);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const unsigned pos0 = kt * kTcKeys, left = static_cast<unsigned>(u.seq.len) - pos0;
                const unsigned boxes = (min(left, static_cast<unsigned>(kTcKeys)) + box_rows - 1) / box_rows;
                if (lane == 0) {
                    mbar_expect_tx(kfull(st), boxes * box_rows * 128 * S::kSubs);
                    mbar_expect_tx(vfull(st), boxes * box_rows * 128 * S::kSubs);
                }
                __syncwarp();
                if (lane < boxes) {
                    const unsigned pos = pos0 + lane * box_rows;
                    const int y = static_cast<int>((tree_page(a, u.seq.slot, pos >> a.page_shift) << a.page_shift) + (pos & (a.page_rows - 1)));
                    const int x = static_cast<int>(u.kv_head * HD);
                    const uint32_t k_at = smem + S::kTile + st * 2 * S::kTile + lane * box_rows * 128, v_at = k_at + S::kTile;
#pragma unroll
                    for (int s = 0; s < S::kSubs; s++) tma_load_2d(k_at + s * S::kPanel, &map_k, x + s * 64, y, kfull(st));
#pragma unroll
                    for (int s = 0; s < S::kSubs; s++) tma_load_2d(v_at + s * S::kPanel, &map_v, x + s * 64, y, vfull(st));
                }
                __syncwarp();
            }
        }
        if (!ok) {
            // what is in flight lands before the CTA gives its memory back
            for (int st = 0; st < S::kStages; st++) {
                const unsigned n = t > static_cast<unsigned>(st) ? (t - 1 - st) / S::kStages : 0u;
                if (t > static_cast<unsigned>(st)) {
                    mbar_wait_bounded(kfull(st), n & 1u, a.wait_limit);
                    mbar_wait_bounded(vfull(st), n & 1u, a.wait_limit);
                }
            }
        }
    } else if (warp == 9) {
        // ---- products ----
        if (lane == 0) {
            constexpr unsigned fmt = std::is_same<T, __half>::value ? 0u : 1u;
            constexpr uint32_t id_s = tc_idesc(fmt, kTcKeys, 0), id_o = tc_idesc(fmt, HD, 1);
            unsigned t = 0, units = 0, ended = 0;  // tiles, blocks begun, blocks whose last product has been issued
            bool first[2] = {true, true};
            // O += P V of tile x
            auto product_v = [&](unsigned x, bool last) -> bool {
                const unsigned w = x & 1u;
                const int st = static_cast<int>(x % S::kStages);
                if (!tc_wait(vfull(st), (x / S::kStages) & 1u, a.wait_limit, gave_up)) return false;
                if (!tc_wait(pready + 8 * w, (x >> 1) & 1u, a.wait_limit, gave_up)) return false;
                tc_fence_after();
                const uint32_t v_at = smem + S::kTile + st * 2 * S::kTile + S::kTile;
#pragma unroll
                for (int k = 0; k < kTcKeys / 16; k++)
                    tc_mma_ts(tmem + 256 + w * HD, tmem + w * 128 + k * 8, tc_desc(v_at + k * 2048, S::kPanel), id_o, !(first[w] && k == 0));
                first[w] = false;
                tc_commit(empty(st));
                if (last) {
                    tc_commit(udone);
                    ended++;
                }
                return true;
            };
            while (ok && walk.next(a, u)) {
                if (t) ok = product_v(t - 1, true);
                first[0] = first[1] = true;
                if (ok) ok = tc_wait(qfull, units & 1u, a.wait_limit, gave_up);
                units++;
                for (unsigned kt = u.k0; ok && kt < u.k1; kt++, t++) {
                    const int st = static_cast<int>(t % S::kStages);
                    ok = tc_wait(kfull(st), (t / S::kStages) & 1u, a.wait_limit, gave_up);
                    // Products of one shape run in the order of their issue, so this one comes after the product that
                    // reads the weights it overwrites; of two shapes that is not said, and the earlier one is waited for.
                    if (HD != 128 && ok && t >= 2) ok = tc_wait(empty(static_cast<int>((t - 2) % S::kStages)), ((t - 2) / S::kStages) & 1u, a.wait_limit, gave_up);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t k_at = smem + S::kTile + st * 2 * S::kTile;
#pragma unroll
                    for (int k = 0; k < HD / 16; k++) {
                        const unsigned off = (k / 4) * S::kPanel + (k % 4) * 32;
                        tc_mma_ss(tmem + (t & 1u) * 128, tc_desc(smem + off, 16), tc_desc(k_at + off, 16), id_s, k != 0);
                    }
                    tc_commit(sfull + 8 * (t & 1u));
                    if (kt > u.k0) ok = product_v(t - 1, false);
                }
            }
            if (ok && t) ok = product_v(t - 1, true);
            if (!ok && t) {
                // the products in flight end before TMEM is given back
                tc_commit(udone);
                mbar_wait_bounded(udone, ended & 1u, a.wait_limit);
            }
        }
        __syncwarp();
    } else {
        // ---- softmax ----
        const unsigned w = warp >> 2, row = tid & 127u;
        const uint32_t lanes = (warp & 3u) << 21;  // the warp's 32 lanes of TMEM
        const uint32_t s_at = tmem + w * 128 + lanes, o_at = tmem + 256 + w * HD + lanes;
        const float scale = fabsf(a.scale_log2);
        const uint32_t flip = a.scale_log2 < 0.0f ? 0x80008000u : 0u;  // a negative scale turns q's sign
        auto load_q = [&](const TreeUnit& x) {
            const unsigned flat0 = x.block * kTcRows, rows_all = x.seq.n * a.group;
#pragma unroll 4
            for (unsigned e = tid; e < 128u * HD / 8; e += kSoftmaxThreads) {
                const unsigned r = e / (HD / 8), c = e % (HD / 8);
                uint4 v = make_uint4(0u, 0u, 0u, 0u);
                if (flat0 + r < rows_all) {
                    const unsigned flat = flat0 + r, node = flat / a.group, head = x.kv_head * a.group + flat % a.group;
                    v = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + static_cast<size_t>(x.seq.row0 + node) * a.q_stride + static_cast<size_t>(head) * HD + c * 8);
                    v.x ^= flip, v.y ^= flip, v.z ^= flip, v.w ^= flip;
                }
                *reinterpret_cast<uint4*>(tc_smem + (c / 8) * S::kPanel + r * 128 + (((c % 8) ^ (r & 7u)) << 4)) = v;
            }
            proxy_fence();
            mbar_arrive(qfull);
        };
        unsigned t = 0, units = 0;
        bool have = ok && walk.next(a, u);
        if (have) load_q(u);
        while (have) {
            const unsigned flat0 = u.block * kTcRows, m_rows = min(static_cast<unsigned>(kTcRows), u.seq.n * a.group - flat0);
            const bool busy = (warp & 3u) * 32 < m_rows;  // some row of the warp is there
            const unsigned flat = flat0 + min(row, m_rows - 1), node = flat / a.group;
            float m = -INFINITY, l = 0.0f;
            bool begun = false;  // a tile of this stream has gone into the accumulator
            for (unsigned kt = u.k0; ok && kt < u.k1; kt++, t++) {
                if ((t & 1u) != w) continue;
                ok = __all_sync(0xffffffffu, tc_wait(sfull + 8 * w, (t >> 1) & 1u, a.wait_limit, gave_up));
                if (!ok) break;
                tc_fence_after();
                const int pos0 = static_cast<int>(kt) * kTcKeys;
                const bool masked = pos0 + kTcKeys > u.seq.ctx;  // drafted rows, or the end, are in the tile
                if (busy) {
                    unsigned bits[4];
                    if (masked) {
#pragma unroll
                        for (int j = 0; j < 4; j++) bits[j] = tree_visible(a, u.seq, node, pos0 + 32 * j);
                    }
                    uint32_t v[32];
                    float top = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        tc_ld32(s_at + 32 * j, v);
                        tc_wait_ld();
                        if (masked) {
#pragma unroll
                            for (int i = 0; i < 32; i++) top = (bits[j] >> i) & 1u ? fmaxf(top, __uint_as_float(v[i])) : top;
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; i++) top = fmaxf(top, __uint_as_float(v[i]));
                        }
                    }
                    if (top != -INFINITY) top *= scale;
                    const float before = m;
                    if (!begun) {
                        m = top;
                    } else if (__any_sync(0xffffffffu, top > m + 8.0f)) {
                        m = fmaxf(m, top);
                        const float f = before == -INFINITY ? 0.0f : ex2(before - m);
                        l *= f;
#pragma unroll
                        for (int j = 0; j < HD / 32; j++) {
                            tc_ld32(o_at + 32 * j, v);
                            tc_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; i++) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
                            tc_st32(o_at + 32 * j, v);
                        }
                    }
                    const float ref = m == -INFINITY ? 0.0f : m;
                    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        tc_ld32(s_at + 32 * j, v);
                        tc_wait_ld();
                        uint32_t p[16];
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            float lo = ex2(fmaf(__uint_as_float(v[2 * i]), scale, -ref)), hi = ex2(fmaf(__uint_as_float(v[2 * i + 1]), scale, -ref));
                            if (masked) {
                                lo = (bits[j] >> (2 * i)) & 1u ? lo : 0.0f;
                                hi = (bits[j] >> (2 * i + 1)) & 1u ? hi : 0.0f;
                            }
                            sum[i & 3] += lo + hi;
                            p[i] = pack2<T>(lo, hi);
                        }
                        tc_st16(s_at + 16 * j, p);
                    }
                    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    tc_wait_st();
                }
                begun = true;
                if (masked) {
                    // V rows behind the last position are cleared (they may hold anything, and 0 * NaN is NaN); so are drafted
                    // ones with an infinity or a NaN, which rows that do not see them must not get: add_bad_values
                    const int st = static_cast<int>(t % S::kStages);
                    ok = __all_sync(0xffffffffu, tc_wait(vfull(st), (t / S::kStages) & 1u, a.wait_limit, gave_up));
                    unsigned char* v_at = tc_smem + S::kTile + st * 2 * S::kTile + S::kTile;
                    const int valid = min(kTcKeys, u.seq.len - pos0), drafted = max(0, u.seq.ctx - pos0);
                    const unsigned quads = S::kSubs * 8;  // 16-byte pieces of a row
                    for (unsigned e = row; ok && e < (kTcKeys - valid) * quads; e += 128) {
                        const unsigned r = valid + e / quads, c = e % quads;
                        *reinterpret_cast<uint4*>(v_at + (c / 8) * S::kPanel + r * 128 + (c % 8) * 16) = make_uint4(0u, 0u, 0u, 0u);
                    }
                    // eight threads to a panel row: a row is cleared by the threads that read it
                    const unsigned g8 = row >> 3, c8 = row & 7u;
                    for (int r0 = drafted; r0 < valid; r0 += 16) {
                        const int r = r0 + static_cast<int>(g8);
                        bool bad = false;
                        if (ok && r < valid) {
#pragma unroll
                            for (int s = 0; s < S::kSubs; s++) {
                                const uint4 x = *reinterpret_cast<const uint4*>(v_at + s * S::kPanel + r * 128 + c8 * 16);
                                bad = bad || bad_pair<T>(x.x) || bad_pair<T>(x.y) || bad_pair<T>(x.z) || bad_pair<T>(x.w);
                            }
                        }
                        const unsigned who = __ballot_sync(0xffffffffu, bad);
                        if (who == 0) continue;
                        if ((who >> (lane & 24u)) & 0xffu) {
#pragma unroll
                            for (int s = 0; s < S::kSubs; s++) *reinterpret_cast<uint4*>(v_at + s * S::kPanel + r * 128 + c8 * 16) = make_uint4(0u, 0u, 0u, 0u);
                            misc[2 + (units & 1u)] = 1;
                        }
                    }
                    proxy_fence();
                }
                tc_fence_before();
                mbar_arrive(pready + 8 * w);
            }
            // every S of the unit has been read, so Q is free
            bar_softmax();
            const TreeUnit done = u;
            have = walk.next(a, u);
            if (have) load_q(u);
            ok = ok && tc_wait(udone, units & 1u, a.wait_limit, gave_up);
            tc_fence_after();
            ml[w * 128 + row] = make_float2(m, l);
            bar_softmax();
            const bool fix = misc[2 + (units & 1u)] != 0;
            const float2 other = ml[(w ^ 1u) * 128 + row];
            // the two streams together: weights of each accumulator, 0 for one that saw nothing (it may never have been written)
            const float top = fmaxf(m, other.x), ref = top == -INFINITY ? 0.0f : top;
            const float f_own = l == 0.0f ? 0.0f : ex2(m - ref), f_other = other.y == 0.0f ? 0.0f : ex2(other.x - ref);
            const float total = (l == 0.0f ? 0.0f : l * f_own) + (other.y == 0.0f ? 0.0f : other.y * f_other);
            const float inv = total == 0.0f ? 0.0f : 1.0f / total;
            if (busy) {
                const unsigned head = done.kv_head * a.group + flat % a.group;
                T* out = static_cast<T*>(a.out) + static_cast<size_t>(done.seq.row0 + node) * a.out_stride + static_cast<size_t>(head) * HD;
                const size_t piece = ((static_cast<size_t>(blockIdx.x) * 2 + done.piece) * kTcRows + row);
                float* po = a.part_o + piece * HD;
                const unsigned c0 = w * (HD / 2);
#pragma unroll
                for (int j = 0; j < HD / 64; j++) {
                    uint32_t x[32], y[32];
                    tc_ld32(tmem + 256 + w * HD + lanes + c0 + 32 * j, x);
                    tc_ld32(tmem + 256 + (w ^ 1u) * HD + lanes + c0 + 32 * j, y);
                    tc_wait_ld();
                    float o[32];
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        o[i] = fmaf(l == 0.0f ? 0.0f : __uint_as_float(x[i]), f_own, other.y == 0.0f ? 0.0f : __uint_as_float(y[i]) * f_other);
                    if (row < m_rows) {
                        if (done.whole) {
#pragma unroll
                            for (int i = 0; i < 32; i += 8)
                                *reinterpret_cast<uint4*>(out + c0 + 32 * j + i) =
                                    make_uint4(pack2<T>(o[i] * inv, o[i + 1] * inv), pack2<T>(o[i + 2] * inv, o[i + 3] * inv),
                                               pack2<T>(o[i + 4] * inv, o[i + 5] * inv), pack2<T>(o[i + 6] * inv, o[i + 7] * inv));
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; i += 4)
                                *reinterpret_cast<float4*>(po + c0 + 32 * j + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                        }
                    }
                }
                if (row < m_rows) {
                    if (!done.whole && w == 0) a.part_ml[piece] = make_float2(top, total);
                    if (fix && total != 0.0f) add_bad_values<T, HD>(a, done, node, head, ref, total, out, done.whole ? nullptr : po, c0, c0 + HD / 2);
                }
            }
            tc_fence_before();
            if (tid == 0) misc[2 + ((units + 1) & 1u)] = 0;  // read a unit ago, written again only behind the barrier
            bar_softmax();
            units++;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (tid == 0 && *gave_up) atomicOr(a.err_word, kErrTimeout);
    if (warp == 8) tc_dealloc(tmem, 512);
}

// cuTensorMapEncodeTiled by way of the runtime: the library links no driver library.
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            return static_cast<EncodeTiled>(nullptr);
        }
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

// A store as rows of n_kv_heads * head_dim elements, fetched as boxes of 64 columns by a page (or 128 rows of a larger one).
bool encode_store(CUtensorMap* map, const TreeArgs& a, const char* base, bool half) {
    const EncodeTiled enc = encode_tiled();
    if (!enc) return false;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(a.n_kv_heads) * a.head_dim, static_cast<cuuint64_t>(a.n_pages) << a.page_shift};
    const cuuint64_t strides[1] = {a.row_bytes};
    const cuuint32_t box[2] = {64, a.page_rows < 128 ? a.page_rows : 128}, step[2] = {1, 1};
    return enc(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<char*>(base), dims, strides, box, step,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int HD>
int launch_tc(lokal_cuda_ctx* ctx, cudaStream_t s, const TreeArgs& a) {
    CUtensorMap map_k, map_v;
    constexpr bool half = std::is_same<T, __half>::value;
    if (!encode_store(&map_k, a, a.k, half) || !encode_store(&map_v, a, a.v, half)) return ctx->fail(LOKAL_ERR_CUDA, "tree_attn: a store cannot be described to the copy engine");
    const unsigned shares = static_cast<unsigned>(ctx->sm_count);
    launch_staged(tree_attn_tc_kernel<T, HD>, shares, kTcThreads, TcShape<HD>::kBytes, s, a, map_k, map_v);
    LOKAL_CHECK_LAUNCH(ctx, "tree_attn_tc_kernel");
    launch_k(tree_join_kernel<T, kTcRows, kTcKeys>, shares - 1, 256, 0, s, a, shares);
    LOKAL_CHECK_LAUNCH(ctx, "tree_join_kernel");
    return LOKAL_OK;
}

}  // namespace

size_t tree_tc_rows(const lokal_cuda_ctx* ctx) { return static_cast<size_t>(ctx->sm_count) * 2 * kTcRows; }

bool tree_tc_takes(const TreeArgs& a, int dtype, int kv_dtype) {
    return dtype == kv_dtype && dtype != LOKAL_F32 && (a.head_dim == 64 || a.head_dim == 128) && a.row_bytes % 16 == 0 && aligned_to(a.k, 16) &&
           aligned_to(a.v, 16) && aligned_to(a.q, 16) && aligned_to(a.out, 16) && a.q_stride % 8 == 0 && a.out_stride % 8 == 0;
}

int launch_tree_tc(lokal_cuda_ctx* ctx, cudaStream_t s, const TreeArgs& a, int dtype) {
    if (dtype == LOKAL_F16) return a.head_dim == 64 ? launch_tc<__half, 64>(ctx, s, a) : launch_tc<__half, 128>(ctx, s, a);
    return a.head_dim == 64 ? launch_tc<__nv_bfloat16, 64>(ctx, s, a) : launch_tc<__nv_bfloat16, 128>(ctx, s, a);
}

}  // namespace lokal
