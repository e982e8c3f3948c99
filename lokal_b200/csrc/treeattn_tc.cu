// Attention of drafted rows over a paged cache on the tensor cores: 16-bit rows of the cache's own type, head sizes 64
// and 128. The other types and shapes run in treeattn.cu; the mathematics and the walk over the work are in treeattn.cuh.
//
// Bound by memory up to about 250 query rows per key head (a key and its value are 4 * head_dim bytes and cost
// 4 * head_dim flops per row; the measured 1634 TFLOP/s over 6570 GB/s are 249 flops per byte), so the aim is that the
// copies never wait. One CTA per SM, 128 query rows by 128 keys:
//   warp 8       brings K tiles, page by page, into a ring with TMA (128-byte swizzle)
//   warp 9       issues S = Q K^T into TMEM
//   warp 10      issues O += P V, with P read from TMEM and V as it lies (MN-major)
//   warp 11      loads the query rows of the next block once the last scores of this one are there, and brings V tiles
//   warps 0-3    take the even tiles, warps 4-7 the odd ones: S from TMEM, maximum, exp2, P back over S
// The two groups of warps are two streams of the running softmax, each with a maximum, a sum and an accumulator of its
// own, so neither waits for the other; they are put together when the block ends. With head size 64, TMEM has room for a
// third S, and the scores of a tile are ready when its group has done the one before; with 128 it is two. The end of a
// block (its last products, then the way out) is hidden behind the scores of the next block's first tiles. The two kinds
// of products have a warp each because issuing them is what costs: one warp for both took 2150 clocks a tile of head size
// 64, half as much again as the copy of the tile. So have the copies: a tile's boxes took one warp 600 clocks for K, 600 for V.
// K and V tiles have their places in one ring in the order of their use.
// A block of up to 16 rows (single tokens, small trees) wastes a tile of 128: every score costs its exponential, and the
// warps whose lanes hold the rows compute 128 keys by 32 rows in turn. With head size 64, and where sequences have few rows on
// average, such blocks are taken by the softmax warps themselves: products of 16 rows by 32 keys a warp, from the same ring,
// every key's weight in a thread of its own (few_rows). Single tokens of 256 sequences of up to 4,096 keys, 32 heads over 4:
// 171 us without it, 144 with it; 8 of 131,072 keys: 206 and 185 (5.8 TB/s). What it costs: blocks end slower (one key tile to
// a sequence: 46 us without it, 50 to 52 with it), larger blocks in the same call run 6 % slower, and with head size 128, where a
// tile's copy takes twice the time, it won 3 % at best and lost 25 % at short lengths, so those keep to the other way.
// An accumulator is rescaled only when the maximum has grown by more than 2^lag since it was last set, so that most tiles
// leave it alone. A row's reference moves by its own scores only: the warp's other rows may be another sequence's, or what an
// earlier call left in the tile. Weights are rounded to the cache's type for the product (half a step each, as the values they multiply
// were); sums, maxima and scores are f32. bf16 has the exponents of f32 and takes weights of up to 2^8 and down to 2^-126. f16
// loses bits below 2^-14, so there weights are taken times 2^11 with a lag of 2^4 (at most 2^15): half a step each down to
// 2^-25 of the largest, and 2^-36 of it below that, where 100,000 keys of 2^-25 are 0.3 % of a row. Sums and accumulators
// carry the factor, the division takes it out.
#include <cuda.h>

#include <type_traits>

#include "treeattn.cuh"

namespace lokal {
namespace {

constexpr unsigned kMaxShares = 512;  // CTAs of the attention kernel, one per SM: more are not used
constexpr int kTcRows = 128, kTcKeys = 128, kTcThreads = 384;
constexpr unsigned kFewRows = 16;  // blocks of up to so many rows take the products of a warp

template <int HD>
struct TcShape {
    static constexpr int kSubs = HD / 64;             // 64-column panels of 128 bytes
    static constexpr unsigned kPanel = 128 * 128;     // bytes of a panel of 128 rows
    static constexpr unsigned kTile = kSubs * kPanel; // bytes of a K or V tile, and of Q
    static constexpr unsigned kSlots = HD == 128 ? 5 : 10;  // K and V tiles in the ring: 160 KB beside two Q tiles
    static constexpr unsigned kScores = HD == 128 ? 2 : 3;  // S tiles in TMEM: 128 columns each, beside two accumulators of HD
    static constexpr unsigned kAhead = kScores - 1;         // tiles whose scores are computed before a tile's output product
    static constexpr unsigned kUnits = 8;  // blocks that the scores may be ahead of the last one written out: four at most
    static constexpr unsigned kRing = 2 * kTile;
    static constexpr unsigned kMl = kRing + kSlots * kTile;  // float2[2][128]
    static constexpr unsigned kBars = kMl + 2 * 128 * 8;     // mbarriers
    static constexpr unsigned kNumBars = 2 * kSlots + 3 * kScores + 5 + kUnits + 1;
    static constexpr unsigned kMisc = kBars + (kNumBars + 1) / 2 * 16;  // TMEM address, flags
    static constexpr unsigned kKnown = kMisc + 32;                      // sequences of the walk
    static constexpr unsigned kUnit = kKnown + kTreeKnown * 16;         // blocks, for the softmax groups
    static constexpr unsigned kBytes = kUnit + kUnits * 32;
    static_assert(kBytes <= 227 * 1024, "a CTA's shared memory");
    static_assert(kScores * 128 + 2 * HD <= 512, "TMEM columns");
};

// Where the barriers are.
template <int HD>
struct TcBars {
    using S = TcShape<HD>;
    uint32_t at;
    __device__ __forceinline__ uint32_t full(unsigned slot) const { return at + slot * 8; }
    __device__ __forceinline__ uint32_t empty(unsigned slot) const { return at + (S::kSlots + slot) * 8; }
    __device__ __forceinline__ uint32_t sfull(unsigned b) const { return at + (2 * S::kSlots + b) * 8; }                    // scores are there
    __device__ __forceinline__ uint32_t pready(unsigned b) const { return at + (2 * S::kSlots + S::kScores + b) * 8; }      // weights are there
    __device__ __forceinline__ uint32_t sfree(unsigned b) const { return at + (2 * S::kSlots + 2 * S::kScores + b) * 8; }   // weights have been used
    __device__ __forceinline__ uint32_t qfull() const { return at + (2 * S::kSlots + 3 * S::kScores) * 8; }                 // Q tiles 0 and 1 each; qfree behind
    __device__ __forceinline__ uint32_t udone() const { return qfull() + 32; }                                              // the last product of a block
    __device__ __forceinline__ uint32_t ufull() const { return udone() + 8; }                                               // a block is described
    __device__ __forceinline__ uint32_t fbar() const { return ufull() + 8 * S::kUnits; }                                    // the softmax groups meet
};

// A slot of the ring and the parity of its round.
template <int HD>
struct RingAt {
    unsigned slot = 0, round = 0;
    __device__ __forceinline__ void skip(unsigned k) {  // any number
        round ^= k / TcShape<HD>::kSlots & 1u;
        add(k % TcShape<HD>::kSlots);
    }
    __device__ __forceinline__ void add(unsigned k) {  // at most a round
        slot += k;
        if (slot >= TcShape<HD>::kSlots) {
            slot -= TcShape<HD>::kSlots;
            round ^= 1u;
        }
    }
};

// Place of a block's tiles in the order of their use, counted from the block's first: K of the first kAhead tiles, then K of
// each further tile and V of the one kAhead before it, then the V tiles that are left.
template <int HD>
__device__ __forceinline__ unsigned v_place(unsigned i, unsigned n) {
    return min(i + TcShape<HD>::kAhead + 1u, n) + i;
}
template <int HD>
__device__ __forceinline__ unsigned k_place(unsigned i) {
    return i + (i > TcShape<HD>::kAhead ? i - TcShape<HD>::kAhead : 0u);
}

// Rows of a block.
__device__ __forceinline__ unsigned rows_of(const TreeArgs& a, unsigned drafted, unsigned block) { return min(a.block_rows, drafted * a.group - block * a.block_rows); }

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
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// One lane of a warp, always the same.
__device__ __forceinline__ bool tc_elect() {
    unsigned yes;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(yes));
    return yes != 0;
}

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
// Waits for the warp's loads; naming the registers keeps their uses behind it.
#define TC_RW4(v, i) "+r"(v[i]), "+r"(v[i + 1]), "+r"(v[i + 2]), "+r"(v[i + 3])
__device__ __forceinline__ void tc_wait_ld(uint32_t (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : TC_RW4(v, 0), TC_RW4(v, 4), TC_RW4(v, 8), TC_RW4(v, 12), TC_RW4(v, 16), TC_RW4(v, 20), TC_RW4(v, 24), TC_RW4(v, 28)
                 :
                 : "memory");
}
__device__ __forceinline__ void tc_ld16(uint32_t at, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : TC_R4(v, 0), TC_R4(v, 4), TC_R4(v, 8), TC_R4(v, 12)
        : "r"(at));
}
__device__ __forceinline__ void tc_wait_ld16(uint32_t (&v)[16], uint32_t (&w)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : TC_RW4(v, 0), TC_RW4(v, 4), TC_RW4(v, 8), TC_RW4(v, 12), TC_RW4(w, 0), TC_RW4(w, 4), TC_RW4(w, 8), TC_RW4(w, 12)
                 :
                 : "memory");
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

// ---- products of a warp (blocks of few rows) ----
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : TC_R4(r, 0) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : TC_R4(r, 0) : "r"(at) : "memory");
}
// c += a b over a contraction of 16: a 16 x 16, b 16 x 8
template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (std::is_same<T, __half>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : TC_W4(a, 0), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : TC_W4(a, 0), "r"(b0), "r"(b1));
}
// A 16-byte piece of a tile in shared memory: panels of 64 columns, rows of 128 bytes, the 128-byte swizzle.
__device__ __forceinline__ uint32_t piece_of(uint32_t tile, unsigned row, unsigned chunk) {
    return tile + (chunk >> 3) * (128u * 128u) + row * 128u + (((chunk ^ row) & 7u) << 4);
}

__device__ __forceinline__ void mbar_arrive_n(uint32_t mbar, unsigned n) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(mbar), "r"(n) : "memory"); }
__device__ __forceinline__ void mbar_arrive(uint32_t mbar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(mbar) : "memory"); }
__device__ __forceinline__ bool mbar_is_done(uint32_t mbar, unsigned parity) {  // a look, without waiting
    unsigned yes;
    asm volatile("{\n.reg .pred p;\nmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(yes) : "r"(mbar), "r"(parity) : "memory");
    return yes != 0;
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t mbar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(mbar)
                 : "memory");
}
__device__ __forceinline__ float ex2(float x) {  // 2 steps of error, 0 for results below the smallest normal value
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// How far the maximum may grow before an accumulator is rescaled, and the factor of weights, as powers of 2.
template <typename T>
struct Weights {
    static constexpr bool kHalf = std::is_same<T, __half>::value;
    static constexpr float kLag = kHalf ? 4.0f : 8.0f, kUp = kHalf ? 11.0f : 0.0f;
};

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
// the two values, 0 for one that is an infinity or a NaN
template <typename T>
__device__ __forceinline__ uint32_t finite_pair(uint32_t v) {
    constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    return ((v & e) == e ? 0u : v & 0xffffu) | (((v >> 16) & e) == e ? 0u : v & 0xffff0000u);
}
// Eight values in shared memory without their infinities and NaNs; whether there were any.
template <typename T>
__device__ __forceinline__ bool make_finite(uint4* p) {
    const uint4 x = *p, y = make_uint4(finite_pair<T>(x.x), finite_pair<T>(x.y), finite_pair<T>(x.z), finite_pair<T>(x.w));
    if (x.x == y.x && x.y == y.y && x.z == y.z && x.w == y.w) return false;
    *p = y;
    return true;
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t mbar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(mbar)
                 : "memory");
}

__device__ __forceinline__ void tma_prefetch(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }

constexpr unsigned kDrainPolls = 1u << 14;  // for what is in flight when a wait has given up: it lands in microseconds

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

// Sixteen 16-bit values of a row: a whole 32-byte sector where the rows allow it.
__device__ __forceinline__ void st_row16(void* p, const uint32_t (&h)[8], bool vec32) {
    if (vec32) {
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), TC_W4(h, 0), TC_W4(h, 4) : "memory");
    } else {
        static_cast<uint4*>(p)[0] = make_uint4(h[0], h[1], h[2], h[3]);
        static_cast<uint4*>(p)[1] = make_uint4(h[4], h[5], h[6], h[7]);
    }
}

// Pieces are kept by column, the rows of a column side by side: the 32 threads that hold 32 rows of an accumulator write
// 128 bytes at a time (by row they wrote 16 bytes each to 32 lines: 8,000 clocks for a piece of 128 x 128, now 2,000).
__device__ __forceinline__ size_t piece_at(size_t piece, unsigned head_dim, unsigned col, unsigned row) {
    return (piece * head_dim + col) * kTcRows + row;
}

// A block as the softmax groups need it, in shared memory; n == 0 ends the walk.
struct __align__(16) TcUnit {
    unsigned row0, len, block_piece, kv_head;  // block * 4 + whole * 2 + piece: of 2^31 rows there are less than 2^25 blocks
    unsigned k0, n;         // key tiles k0 .. k0 + n
    unsigned drafted;       // drafted rows of the sequence
    unsigned slot;
    __device__ int ctx() const { return static_cast<int>(len - drafted); }
    __device__ unsigned block() const { return block_piece >> 2; }
    __device__ bool whole() const { return (block_piece & 2u) != 0; }
    __device__ unsigned piece() const { return block_piece & 1u; }
};

// Infinities and NaNs in V rows of drafted rows were set to 0 for the product, because rows that do not
// see them would get 0 * inf. What they add to the rows that do see them is added here, to the stored result: rare, and
// slow (a dot product per row and value).
template <typename T, int HD>
__device__ __noinline__ void add_bad_values(const TreeArgs& a, const TcUnit* unit, unsigned node, unsigned head, float m, float l, T* out, float* piece,
                                            unsigned c0, unsigned c1) {
    const TreeSeq seq{unit->row0, unit->drafted, unit->ctx(), static_cast<int>(unit->len), unit->slot};
    const int first = max(seq.ctx, static_cast<int>(unit->k0) * kTcKeys), last = min(seq.len, static_cast<int>(unit->k0 + unit->n) * kTcKeys);
    const T* q = static_cast<const T*>(a.q) + static_cast<size_t>(seq.row0 + node) * a.q_stride + static_cast<size_t>(head) * HD;
    for (int pos = first; pos < last; pos++) {
        if (!(tree_visible(a, seq, node, pos) & 1u)) continue;
        const size_t row = (static_cast<size_t>(tree_page(a, seq.slot, static_cast<unsigned>(pos) >> a.page_shift)) << a.page_shift) +
                           (static_cast<unsigned>(pos) & (a.page_rows - 1));
        const size_t off = row * a.row_bytes + static_cast<size_t>(unit->kv_head) * HD * 2;
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
                p = exp2f(fmaf(s, a.scale_log2, Weights<T>::kUp - m));
                have = true;
            }
            if (piece) piece[static_cast<size_t>(c) * kTcRows] += p * x;
            else out[c] = from_f32<T>(to_f32<T>(out[c]) + p * x / l);
        }
    }
}

// A block of few rows, without TMEM: the groups take its tiles in turn and a warp 32 keys of a tile, with sums, maxima and an
// output of its own. (All warps on every tile, 16 keys each: 10 us more at 256 sequences.)
template <typename T, int HD>
__device__ __forceinline__ bool few_rows(const TreeArgs& a, const TcUnit* now, unsigned units, unsigned ring_t, unsigned met, bool ok) {
    using S = TcShape<HD>;
    extern __shared__ __align__(1024) unsigned char tc_smem[];
    const uint32_t smem = smem_addr(tc_smem), bars = smem + S::kBars;
    const unsigned tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, w = warp >> 2;
    const TcBars<HD> at_bar{bars};
    volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(tc_smem + S::kMisc);
    volatile int* gave_up = reinterpret_cast<volatile int*>(misc + 1);
    float2* ml = reinterpret_cast<float2*>(tc_smem + S::kMl);
    const float scale = a.scale_log2;
    const auto full = [&](unsigned slot) { return at_bar.full(slot); };
    const auto empty = [&](unsigned slot) { return at_bar.empty(slot); };
    const uint32_t qfull = at_bar.qfull(), qfree = qfull + 16, fbar = at_bar.fbar();
    const auto look = [&](unsigned slot, unsigned round) {
        ok = ok && __all_sync(0xffffffffu, tc_wait(full(slot), round, a.wait_limit, gave_up));
        if (ok && lane == 0) mbar_arrive(empty(slot));
        __syncwarp();
    };
    const auto meet = [&] {
        __syncwarp();
        if (lane == 0) mbar_arrive(fbar);
        ok = __all_sync(0xffffffffu, tc_wait(fbar, met, a.wait_limit, gave_up)) && ok;
        met ^= 1u;
    };
    const unsigned n = now->n, qb = units & 1u, g = lane >> 2, c = lane & 3u, pair = warp & 3u;
    const unsigned flat0 = now->block() * a.block_rows, m_rows = rows_of(a, now->drafted, now->block());
    const int len = static_cast<int>(now->len), ctx = now->ctx();
    const TreeSeq seq{now->row0, now->drafted, ctx, len, 0u};
    unsigned node[2];  // of rows g and g + 8
    unsigned long long words[2][2] = {{0ull, 0ull}, {0ull, 0ull}};
    const bool has_mask = a.mask && static_cast<int>((now->k0 + n) * kTcKeys) > ctx;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        node[h] = (flat0 + min(g + 8 * h, m_rows - 1)) / a.group;
        if (has_mask) {
            const unsigned long long* mask = a.mask + static_cast<size_t>(now->row0 + node[h]) * a.mask_words;
            words[h][0] = mask[0];
            if (a.mask_words > 1) words[h][1] = mask[1];
        }
    }
    ok = __all_sync(0xffffffffu, ok && tc_wait(qfull + 8 * qb, (units >> 1) & 1u, a.wait_limit, gave_up));
    uint32_t q[HD / 16][4];
#pragma unroll
    for (int s = 0; s < HD / 16; s++) ldsm4(q[s], piece_of(smem + qb * S::kTile, lane & 15u, 2 * s + (lane >> 4)));
    meet();  // all have the query rows: their tile is where the sums are put together
    float o[HD / 8][4];
#pragma unroll
    for (int j = 0; j < HD / 8; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
    float mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
    const auto look_at = [&](unsigned at) { look(at % S::kSlots, (at / S::kSlots) & 1u); };
    for (unsigned i = 0; ok && i < n; i++) {
        const unsigned k_at = 2 * ring_t + k_place<HD>(i), v_at = 2 * ring_t + v_place<HD>(i, n);
        if ((ring_t + i + w) & 1u) {  // the other group's; its V is looked at with this group's next
            look_at(k_at);
            if (i + 1 == n) look_at(v_at);
            continue;
        }
        const unsigned k_slot = k_at % S::kSlots, v_slot = v_at % S::kSlots;
        const uint32_t k_tile = smem + S::kRing + k_slot * S::kTile, v_tile = smem + S::kRing + v_slot * S::kTile;
        const int pos0 = static_cast<int>((now->k0 + i) * kTcKeys + pair * 32);
        ok = __all_sync(0xffffffffu, tc_wait(full(k_slot), (k_at / S::kSlots) & 1u, a.wait_limit, gave_up));
        if (!ok) break;
        float z[4][4];
#pragma unroll
        for (int x = 0; x < 4; x++) z[x][0] = z[x][1] = z[x][2] = z[x][3] = 0.0f;
#pragma unroll
        for (int s = 0; s < HD / 16; s++) {
#pragma unroll
            for (int x = 0; x < 4; x += 2) {
                uint32_t k[4];  // keys 0 - 7 and 8 - 15 of 16, two pieces each
                ldsm4(k, piece_of(k_tile, pair * 32 + x * 8 + (lane >> 4) * 8 + (lane & 7u), 2 * s + ((lane >> 3) & 1u)));
                mma16<T>(z[x], q[s], k[0], k[1]);
                mma16<T>(z[x + 1], q[s], k[2], k[3]);
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty(k_slot));
        const bool masked = pos0 + 32 > ctx;
        if (masked) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const unsigned seen = (seq.n <= 128 ? tree_visible2(a, seq, node[h], pos0, words[h][0], words[h][1]) : tree_visible(a, seq, node[h], pos0)) >> (2 * c);
#pragma unroll
                for (int x = 0; x < 4; x++) {
#pragma unroll
                    for (int e = 0; e < 2; e++) z[x][2 * h + e] = (seen >> (8 * x + e)) & 1u ? z[x][2 * h + e] : -INFINITY;
                }
            }
        }
        float top[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            top[h] = fmaxf(fmaxf(fmaxf(z[0][2 * h], z[0][2 * h + 1]), fmaxf(z[1][2 * h], z[1][2 * h + 1])),
                           fmaxf(fmaxf(z[2][2 * h], z[2][2 * h + 1]), fmaxf(z[3][2 * h], z[3][2 * h + 1])));
            top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
            top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
            if (top[h] != -INFINITY) top[h] *= scale;
        }
        if (__any_sync(0xffffffffu, top[0] > mx[0] + Weights<T>::kLag || top[1] > mx[1] + Weights<T>::kLag)) {
            float f[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const float before = mx[h];
                if (top[h] > before + Weights<T>::kLag) mx[h] = top[h];
                f[h] = before == -INFINITY ? 0.0f : ex2(before - mx[h]);
                sum[h] *= f[h];
            }
#pragma unroll
            for (int j = 0; j < HD / 8; j++) {
#pragma unroll
                for (int e = 0; e < 4; e++) o[j][e] *= f[e >> 1];
            }
        }
        uint32_t p[2][4];  // of 16 keys: weights of keys 2c, 2c + 1 and 2c + 8, 2c + 9, rows g and g + 8
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const float ref = (mx[h] == -INFINITY ? 0.0f : mx[h]) - Weights<T>::kUp;
            float part[2] = {0.0f, 0.0f};
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const float y0 = ex2(fmaf(z[x][2 * h], scale, -ref)), y1 = ex2(fmaf(z[x][2 * h + 1], scale, -ref));
                part[x & 1] += y0 + y1;
                p[x >> 1][2 * (x & 1) + h] = pack2<T>(y0, y1);
            }
            sum[h] += part[0] + part[1];
        }
        if (i) look_at(2 * ring_t + v_place<HD>(i - 1, n));
        ok = __all_sync(0xffffffffu, ok && tc_wait(full(v_slot), (v_at / S::kSlots) & 1u, a.wait_limit, gave_up));
        if (!ok) break;
        if (masked) {
            // as in clear_v, the warp's own 32 rows, four at a time
            for (int r0 = max(0, ctx - pos0) & ~3; r0 < 32; r0 += 4) {
                const int r = r0 + static_cast<int>(lane >> 3), pos = pos0 + r;
                uint4* v = reinterpret_cast<uint4*>(tc_smem + S::kRing + v_slot * S::kTile + (pair * 32 + r) * 128) + (lane & 7u);
#pragma unroll
                for (int e = 0; e < S::kSubs; e++) {
                    if (pos >= len) v[e * (S::kPanel / 16)] = make_uint4(0u, 0u, 0u, 0u);
                    else if (pos >= ctx && make_finite<T>(v + e * (S::kPanel / 16))) misc[2 + (units & 3u)] = 1;
                }
            }
            proxy_fence();
            __syncwarp();
        }
#pragma unroll
        for (int x = 0; x < 2; x++) {
#pragma unroll
            for (int j = 0; j < HD / 16; j++) {
                uint32_t v[4];  // columns 16 j .. + 7 and + 8 .. + 15, keys 0 - 7 and 8 - 15 each
                ldsm4_t(v, piece_of(v_tile, pair * 32 + x * 16 + (lane & 15u), 2 * j + (lane >> 4)));
                mma16<T>(o[2 * j], p[x], v[0], v[1]);
                mma16<T>(o[2 * j + 1], p[x], v[2], v[3]);
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty(v_slot));
    }
    // Eight warps' sums to four (warps 4 - 7 leave theirs for warps 0 - 3), then all threads put the four together.
    float* all = reinterpret_cast<float*>(tc_smem + qb * S::kTile);  // [4][16 rows][HD], the columns turned by the row
    const auto place_of = [&](unsigned from, unsigned row, unsigned col) { return (from * 16 + row) * HD + (col ^ ((row & 3u) << 3)); };
#pragma unroll
    for (int h = 0; h < 2; h++) {
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
    }
    const auto leave = [&] {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            if (c == 0) ml[pair * 16 + g + 8 * h] = make_float2(mx[h], sum[h]);
#pragma unroll
            for (int j = 0; j < HD / 8; j++) *reinterpret_cast<float2*>(all + place_of(pair, g + 8 * h, 8 * j + 2 * c)) = make_float2(o[j][2 * h], o[j][2 * h + 1]);
        }
    };
    if (warp >= 4) leave();
    meet();
    const bool fix = misc[2 + (units & 3u)] != 0;
    if (tid == 0) misc[2 + ((units + 2) & 3u)] = 0;
    if (warp < 4) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const float2 other = ml[pair * 16 + g + 8 * h];
            const float both = fmaxf(mx[h], other.x), ref = both == -INFINITY ? 0.0f : both;
            const float f_own = sum[h] == 0.0f ? 0.0f : ex2(mx[h] - ref), f_other = other.y == 0.0f ? 0.0f : ex2(other.x - ref);
#pragma unroll
            for (int j = 0; j < HD / 8; j++) {
                const float2 x = *reinterpret_cast<const float2*>(all + place_of(pair, g + 8 * h, 8 * j + 2 * c));
                o[j][2 * h] = fmaf(o[j][2 * h], f_own, x.x * f_other);
                o[j][2 * h + 1] = fmaf(o[j][2 * h + 1], f_own, x.y * f_other);
            }
            sum[h] = fmaf(sum[h], f_own, other.y * f_other);
            mx[h] = both;
        }
        __syncwarp();
        leave();
    }
    meet();
    const unsigned row = tid & 15u, c0 = (tid >> 4) * (HD / 16);
    if (row < m_rows) {
        const bool whole = now->whole();
        float2 parts[4];
#pragma unroll
        for (int x = 0; x < 4; x++) parts[x] = ml[x * 16 + row];
        const float most = fmaxf(fmaxf(parts[0].x, parts[1].x), fmaxf(parts[2].x, parts[3].x)), ref = most == -INFINITY ? 0.0f : most;
        float total = 0.0f, f[4];
#pragma unroll
        for (int x = 0; x < 4; x++) {
            f[x] = parts[x].y == 0.0f ? 0.0f : ex2(parts[x].x - ref);
            total = fmaf(parts[x].y, f[x], total);
        }
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
        const unsigned flat = flat0 + row, node_r = flat / a.group, head = now->kv_head * a.group + flat % a.group;
        T* out = static_cast<T*>(a.out) + static_cast<size_t>(now->row0 + node_r) * a.out_stride + static_cast<size_t>(head) * HD;
        const unsigned piece = blockIdx.x * 2 + now->piece();
        float* po = a.part_o + piece_at(piece, HD, 0, row);
        float y[HD / 16];
#pragma unroll
        for (int e = 0; e < HD / 16; e++) y[e] = 0.0f;
#pragma unroll
        for (int x = 0; x < 4; x++) {
#pragma unroll
            for (int e = 0; e < HD / 16; e += 4) {
                const float4 v = *reinterpret_cast<const float4*>(all + place_of(x, row, c0 + e));
                y[e] = fmaf(v.x, f[x], y[e]);
                y[e + 1] = fmaf(v.y, f[x], y[e + 1]);
                y[e + 2] = fmaf(v.z, f[x], y[e + 2]);
                y[e + 3] = fmaf(v.w, f[x], y[e + 3]);
            }
        }
        if (whole) {
#pragma unroll
            for (int e = 0; e < HD / 16; e += 4)
                *reinterpret_cast<uint2*>(out + c0 + e) = make_uint2(pack2<T>(y[e] * inv, y[e + 1] * inv), pack2<T>(y[e + 2] * inv, y[e + 3] * inv));
        } else {
#pragma unroll
            for (int e = 0; e < HD / 16; e++) po[static_cast<size_t>(c0 + e) * kTcRows] = y[e];
            if (c0 == 0) a.part_ml[piece * kTcRows + row] = make_float2(most, total);
        }
        if (fix && total != 0.0f) add_bad_values<T, HD>(a, now, node_r, head, ref, total, out, whole ? nullptr : po, c0, c0 + HD / 16);
    }
    proxy_fence();
    __syncwarp();
    if (lane == 0) mbar_arrive(qfree + 8 * qb);
    return ok;
}

// FEW: blocks of few rows take the products of a warp.
template <typename T, int HD, bool FEW>
__global__ void __launch_bounds__(kTcThreads, 1)
    tree_attn_tc_kernel(const __grid_constant__ TreeArgs a, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                        const __grid_constant__ CUtensorMap map_v) {
    using S = TcShape<HD>;
    extern __shared__ __align__(1024) unsigned char tc_smem[];
    const uint32_t smem = smem_addr(tc_smem);
    const unsigned tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const uint32_t bars = smem + S::kBars;
    const TcBars<HD> at_bar{bars};
    const auto full = [&](unsigned slot) { return at_bar.full(slot); };
    const auto empty = [&](unsigned slot) { return at_bar.empty(slot); };
    const auto sfull = [&](unsigned b) { return at_bar.sfull(b); };
    const auto pready = [&](unsigned b) { return at_bar.pready(b); };
    const auto sfree = [&](unsigned b) { return at_bar.sfree(b); };
    const uint32_t qfull = at_bar.qfull(), qfree = qfull + 16, udone = at_bar.udone(), ufull = at_bar.ufull(), fbar = at_bar.fbar();
    volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(tc_smem + S::kMisc);  // [0] TMEM, [1] a wait gave up, [2..5] bad values, by block
    volatile int* gave_up = reinterpret_cast<volatile int*>(misc + 1);
    float2* ml = reinterpret_cast<float2*>(tc_smem + S::kMl);
    // set-up that touches no global memory goes ahead of the wait for the launch before
    if (warp == 8) {
        tc_alloc(smem + S::kMisc, 512);
        if (lane == 0) {
            for (unsigned i = 0; i < 2 * S::kSlots; i++) mbar_init(bars + i * 8, FEW && i >= S::kSlots ? 10 : 1);  // full, empty
            for (unsigned b = 0; b < S::kScores; b++) mbar_init(sfull(b), 1);
            for (unsigned b = 0; b < S::kScores; b++) {
                mbar_init(pready(b), 4);
                mbar_init(sfree(b), 1);
            }
            for (unsigned b = 0; b < 2; b++) {
                mbar_init(qfull + 8 * b, 1);
                mbar_init(qfree + 8 * b, FEW ? 10 : 1);
            }
            mbar_init(udone, 1);
            for (unsigned i = 0; i < S::kUnits; i++) mbar_init(ufull + 8 * i, 1);
            mbar_init(fbar, 8);
            mbar_init_fence();
            for (int i = 1; i < 6; i++) misc[i] = 0;
        }
    }
    if (warp == 9 && lane < 3) tma_prefetch(lane == 0 ? &map_q : lane == 1 ? &map_k : &map_v);
    pdl_wait();
    pdl_launch();  // only now: tree_join_tc_kernel looks at the lengths before it waits for this launch
    // the tile of the first query rows is not in use yet: its first bytes hold the sums of the walk
    const unsigned shares = gridDim.x;
    const TreePlace place = tree_locate<kTcKeys, kTcThreads>(a, reinterpret_cast<unsigned long long*>(tc_smem), blockIdx.x == 0, [&](unsigned total) {
        const TreeShares s(total, shares);
        return blockIdx.x < s.g ? s.first(blockIdx.x) : total;
    });
    int4* known = reinterpret_cast<int4*>(tc_smem + S::kKnown);
    if (warp == 10 && lane < kTreeKnown && place.seq + lane < a.n_seqs) {
        const TreeSeq q = tree_seq(a, place.seq + lane, false);
        known[lane] = make_int4(static_cast<int>(q.row0), static_cast<int>(q.n), q.len, static_cast<int>(q.slot));
    }
    proxy_fence();  // the walk's reads and writes of the tile come before those of the copy engine
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = misc[0];
    const TreeShares share(place.total, shares);
    bool ok = place.seq < a.n_seqs;
    TreeWalk<kTcKeys> walk;
    walk.start(a, place, ok ? share.first(blockIdx.x) : 0u, ok ? share.first(blockIdx.x + 1) : 0u, known);
    TreeUnit u;

    // A wait by parity cannot tell a phase from the one after the next, so a warp that waits for tiles has to have seen each
    // place of the ring filled before it asks for the next filling. Tiles that a warp has no use for it looks on: it waits for
    // them and counts as one of those that empty them.
    const auto look = [&](unsigned slot, unsigned round) {
        ok = ok && __all_sync(0xffffffffu, tc_wait(full(slot), round, a.wait_limit, gave_up));
        if (ok && lane == 0) mbar_arrive(empty(slot));
        __syncwarp();
    };
    const auto look_on = [&](RingAt<HD>& at, unsigned n) {  // a whole block of n tiles
        for (unsigned i = 0; ok && i < n; i++) {
            RingAt<HD> k = at, v = at;
            k.skip(k_place<HD>(i));
            v.skip(v_place<HD>(i, n));
            look(k.slot, k.round);
            look(v.slot, v.round);
        }
        at.skip(2 * n);
    };

    if (warp == 8 || warp == 11) {
        // ---- K tiles (warp 8), query rows and V tiles (warp 11) ----
        const bool is_k = warp == 8;
        const CUtensorMap* map = is_k ? &map_k : &map_v;
        const unsigned box_rows = min(a.page_rows, static_cast<unsigned>(kTcKeys));
        RingAt<HD> at;
        bool reused = false;               // the ring has been round once
        unsigned units = 0, issued = 0, parity = 0;  // blocks; by slot: whether it was filled, and in which round
        // query rows: a walk of its own, a block ahead
        TreeWalk<kTcKeys> q_walk = walk;
        TreeUnit q_unit;
        unsigned q_block = 0, q_blocks = 0;  // the next, and how many have been asked for
        bool q_more = !is_k && ok && q_walk.next(a, q_unit);
        const auto put_q = [&](bool must) {
            const unsigned b = q_block & 1u;
            if (!q_more) {
                q_block = 0xffffffffu;
                return;
            }
            if (q_block >= 2) {
                const unsigned phase = ((q_block >> 1) - 1) & 1u;
                if (must) ok = __all_sync(0xffffffffu, tc_wait(qfree + 8 * b, phase, a.wait_limit, gave_up));
                else if (!__all_sync(0xffffffffu, mbar_is_done(qfree + 8 * b, phase))) return;
                if (!ok) return;
            }
            if (lane == 0) {
                const unsigned nodes = kTcRows / a.group;
                mbar_expect_tx(qfull + 8 * b, nodes * a.group * 128 * S::kSubs);
#pragma unroll
                for (int c = 0; c < S::kSubs; c++)
                    tma_load_3d(smem + b * S::kTile + c * S::kPanel, &map_q, c * 64, static_cast<int>(q_unit.kv_head * a.group), static_cast<int>(q_unit.seq.row0 + q_unit.block * nodes),
                                qfull + 8 * b);
            }
            __syncwarp();
            q_block++;
            q_blocks++;
            q_more = q_walk.next(a, q_unit);
        };
        while (ok && walk.next(a, u)) {
            const unsigned n = u.k1 - u.k0;
            // The block's pages, 32 at a time, a lane each, the next 32 on their way (pages to a tile divide 32, so no tile
            // lies across two batches).
            const unsigned first_page = u.k0 * kTcKeys >> a.page_shift, last_page = (min(u.k1 * kTcKeys, static_cast<unsigned>(u.seq.len)) - 1) >> a.page_shift;
            const auto pages_at = [&](unsigned p) { return p + lane <= last_page ? tree_page(a, u.seq.slot, p + lane) : 0u; };
            unsigned page0 = first_page, pages = pages_at(first_page), pages_next = pages_at(first_page + 32);
            if (!is_k) {
                // this block's query rows unless they are on their way, and the next block's as soon as their tile is free
                while (ok && q_block <= units) put_q(true);
                units++;
            }
            unsigned behind = is_k ? 0u : v_place<HD>(0, n);
            reused |= at.slot + behind >= S::kSlots;
            at.add(behind);
            const int x = static_cast<int>(u.kv_head * HD);
            for (unsigned i = 0; i < n; i++) {
                if (reused) ok = __all_sync(0xffffffffu, tc_wait(empty(at.slot), at.round ^ 1u, a.wait_limit, gave_up));
                if (!ok) break;
                const unsigned left = static_cast<unsigned>(u.seq.len) - (u.k0 + i) * kTcKeys;
                const unsigned boxes = (min(left, static_cast<unsigned>(kTcKeys)) + box_rows - 1) / box_rows;
                issued |= 1u << at.slot;
                parity = (parity & ~(1u << at.slot)) | (at.round << at.slot);
                const unsigned pos = (u.k0 + i) * kTcKeys, page = pos >> a.page_shift;
                if (page - page0 >= 32) {
                    page0 += 32;
                    pages = pages_next;
                    pages_next = pages_at(page0 + 32);
                }
                const unsigned mine = __shfl_sync(0xffffffffu, pages, min(page - page0 + lane, 31u));
                const int y = static_cast<int>((mine << a.page_shift) + (pos & (a.page_rows - 1)));
                if (lane == 0) mbar_expect_tx(full(at.slot), boxes * box_rows * 128 * S::kSubs + a.extra_tx);
                __syncwarp();
                if (lane < boxes) {
                    const uint32_t to = smem + S::kRing + at.slot * S::kTile + lane * box_rows * 128;
#pragma unroll
                    for (int c = 0; c < S::kSubs; c++) tma_load_2d(to + c * S::kPanel, map, x + c * 64, y, full(at.slot));
                }
                if (!is_k && q_block <= units) put_q(false);
                const unsigned next = i + 1 == n ? 2 * n : is_k ? i + 1 + (i + 1 > S::kAhead ? i + 1 - S::kAhead : 0u) : v_place<HD>(i + 1, n);
                reused |= at.slot + (next - behind) >= S::kSlots;
                at.add(next - behind);
                behind = next;
            }
        }
        if (!ok && place.seq < a.n_seqs) {
            // what is in flight lands before the CTA gives its memory back (however soon the wait before gave up)
            for (unsigned slot = 0; slot < S::kSlots; slot++)
                if ((issued >> slot) & 1u) mbar_wait_bounded(full(slot), (parity >> slot) & 1u, kDrainPolls);
            if (!is_k) {
                for (unsigned q = q_blocks > 2 ? q_blocks - 2 : 0u; q < q_blocks; q++) mbar_wait_bounded(qfull + 8 * (q & 1u), (q >> 1) & 1u, kDrainPolls);
            }
        }
    } else if (warp == 9) {
        // ---- S = Q K^T ----
        constexpr uint32_t idesc = tc_idesc(std::is_same<T, __half>::value ? 0u : 1u, kTcKeys, 0);
        const uint64_t q_desc = tc_desc(smem, 16), k_desc = tc_desc(smem + S::kRing, 16);
        RingAt<HD> at;                     // of the next K tile
        unsigned b = 0, b_round = 0, t = 0, units = 0;  // S tile, key tiles, blocks
        bool few = false;                  // the block before was one of few rows
        const auto wait = [&](uint32_t bar, unsigned parity) { ok = ok && __all_sync(0xffffffffu, tc_wait(bar, parity, a.wait_limit, gave_up)); };
        TcUnit* described = reinterpret_cast<TcUnit*>(tc_smem + S::kUnit);
        const auto publish = [&](unsigned n) {  // block `units`, to the softmax groups
            if (lane == 0) {
                described[units % S::kUnits] = TcUnit{u.seq.row0, static_cast<unsigned>(u.seq.len), u.block * 4 + (u.whole ? 2u : 0u) + u.piece, u.kv_head, u.k0, n, u.seq.n, u.seq.slot};
                mbar_arrive(ufull + 8 * (units % S::kUnits));
            }
            __syncwarp();
        };
        while (ok && walk.next(a, u)) {
            const unsigned n = u.k1 - u.k0, qb = units & 1u;
            publish(n);
            wait(qfull + 8 * qb, (units >> 1) & 1u);
            if (FEW && rows_of(a, u.seq.n, u.block) <= kFewRows) {  // the softmax groups do it all
                if (t) wait(sfree((t - 1) % S::kScores), ((t - 1) / S::kScores) & 1u);  // all tiles so far have come, V as well
                look_on(at, n);
                if (ok && lane == 0) mbar_arrive(qfree + 8 * qb);
                __syncwarp();
                few = true;
                units++;
                continue;
            }
            // K tiles are not to be used up here while V tiles of a block of few rows still lie in the ring: the copies of K
            // would run more than a round ahead of those of V.
            if (FEW && few) wait(qfree + 8 * (qb ^ 1u), ((units - 1) >> 1) & 1u);
            few = false;
            for (unsigned i = 0; ok && i < n; i++) {
                wait(full(at.slot), at.round);
                if (t >= S::kScores) wait(sfree(b), b_round ^ 1u);  // the weights that these scores overwrite have been used
                if (!ok) break;
                tc_fence_after();
                if (tc_elect()) {
                    const uint64_t qd = q_desc + qb * (S::kTile >> 4), kd = k_desc + at.slot * (S::kTile >> 4);
#pragma unroll
                    for (int k = 0; k < HD / 16; k++) {
                        const unsigned off = ((k / 4) * S::kPanel + (k % 4) * 32) >> 4;
                        tc_mma_ss(tmem + b * 128, qd + off, kd + off, idesc, k != 0);
                    }
                    tc_commit(sfull(b));
                    tc_commit(empty(at.slot));
                    if (FEW) mbar_arrive_n(empty(at.slot), 9);
                    if (i == n - 1) {
                        tc_commit(qfree + 8 * qb);
                        if (FEW) mbar_arrive_n(qfree + 8 * qb, 9);
                    }
                }
                __syncwarp();
                if (++b == S::kScores) {
                    b = 0;
                    b_round ^= 1u;
                }
                t++;
                at.add(i + 1 < n ? (i < S::kAhead ? 1u : 2u) : n + 1 - (n > S::kAhead + 1 ? n - 1 - S::kAhead : 0u));
            }
            units++;
        }
        if (ok) publish(0);
        if (!ok && place.seq < a.n_seqs) {
            // the products in flight end before TMEM is given back
            if (t) mbar_wait_bounded(sfull((t - 1) % S::kScores), ((t - 1) / S::kScores) & 1u, kDrainPolls);
        }
    } else if (warp == 10) {
        // ---- O += P V ----
        constexpr uint32_t idesc = tc_idesc(std::is_same<T, __half>::value ? 0u : 1u, HD, 1);
        const uint64_t v_desc = tc_desc(smem + S::kRing, S::kPanel);
        RingAt<HD> at;
        unsigned b = 0, b_round = 0, t = 0, units = 0, blocks = 0;  // ..., blocks with products here, all blocks
        const auto wait = [&](uint32_t bar, unsigned parity) { ok = ok && __all_sync(0xffffffffu, tc_wait(bar, parity, a.wait_limit, gave_up)); };
        while (ok && walk.next(a, u)) {
            const unsigned n = u.k1 - u.k0;
            if (FEW && rows_of(a, u.seq.n, u.block) <= kFewRows) {
                look_on(at, n);
                if (ok && lane == 0) mbar_arrive(qfree + 8 * (blocks & 1u));
                __syncwarp();
                blocks++;
                continue;
            }
            blocks++;
            unsigned begun = 0;  // bit w: stream w of the block has something in its accumulator
            unsigned behind = v_place<HD>(0, n);
            at.add(behind);
            for (unsigned i = 0; ok && i < n; i++) {
                wait(full(at.slot), at.round);
                wait(pready(b), b_round);
                if (!ok) break;
                tc_fence_after();
                const unsigned w = t & 1u;
                if (tc_elect()) {
                    const uint64_t vd = v_desc + at.slot * (S::kTile >> 4);
#pragma unroll
                    for (int k = 0; k < kTcKeys / 16; k++)
                        tc_mma_ts(tmem + S::kScores * 128 + w * HD, tmem + b * 128 + k * 8, vd + k * (2048 >> 4), idesc, k != 0 || (begun >> w) & 1u);
                    tc_commit(sfree(b));
                    tc_commit(empty(at.slot));
                    if (FEW) mbar_arrive_n(empty(at.slot), 9);
                    if (i == n - 1) tc_commit(udone);
                }
                __syncwarp();
                begun |= 1u << w;
                if (++b == S::kScores) {
                    b = 0;
                    b_round ^= 1u;
                }
                t++;
                const unsigned next = i + 1 < n ? v_place<HD>(i + 1, n) : 2 * n;
                at.add(next - behind);
                behind = next;
            }
            if (ok) units++;
        }
        if (!ok && place.seq < a.n_seqs) {
            // the products in flight end before TMEM is given back
            if (tc_elect()) tc_commit(udone);
            mbar_wait_bounded(udone, units & 1u, kDrainPolls);
        }
    } else {
        // ---- softmax ----
        const unsigned w = warp >> 2, row = tid & 127u;
        const uint32_t lanes = (warp & 3u) << 21;  // the warp's 32 lanes of TMEM
        const uint32_t o_at = tmem + S::kScores * 128 + lanes;
        const float scale = a.scale_log2;
        // before the block: key tiles (each is two of the ring's) and blocks, all and those with products on the big tensor cores
        unsigned ring_t = 0, units = 0, t = 0, big_units = 0;
        const TcUnit* described = reinterpret_cast<const TcUnit*>(tc_smem + S::kUnit);
        // of the block before this one, which may not have been written yet
        float last_m = 0.0f, last_l = 0.0f;
        bool pending = false;
        // The two groups meet. (A wait that can give up, not a hardware barrier: were one group to
        // give up on something else, the other would stand there for good.)
        unsigned met = 0;
        const auto meet = [&](unsigned phase) {  // twice for every block, unless there are blocks of few rows
            __syncwarp();
            if (lane == 0) mbar_arrive(fbar);
            ok = __all_sync(0xffffffffu, tc_wait(fbar, FEW ? met : phase, a.wait_limit, gave_up)) && ok;
            met ^= 1u;
        };
        // The two streams of a block are put together and written out.
        const auto finish = [&] {
            const unsigned which = units - 1;  // the block's number
            const TcUnit* last = described + which % S::kUnits;
            const bool whole = last->whole();
            const unsigned flat0 = last->block() * a.block_rows, m_rows = rows_of(a, last->drafted, last->block());
            ok = __all_sync(0xffffffffu, ok && tc_wait(udone, (FEW ? big_units - 1 : which) & 1u, a.wait_limit, gave_up));
            tc_fence_after();
            ml[w * 128 + row] = make_float2(last_m, last_l);
            meet(0);
            const bool fix = misc[2 + (which & 3u)] != 0;
            if (tid == 0) misc[2 + ((which + 2) & 3u)] = 0;  // read two blocks ago, written again only behind the barrier below
            const float2 other = ml[(w ^ 1u) * 128 + row];
            // weights of the two accumulators, 0 for one that saw nothing (it may never have been written)
            const float top = fmaxf(last_m, other.x), ref = top == -INFINITY ? 0.0f : top;
            const float f_own = last_l == 0.0f ? 0.0f : ex2(last_m - ref), f_other = other.y == 0.0f ? 0.0f : ex2(other.x - ref);
            const float total = (last_l == 0.0f ? 0.0f : last_l * f_own) + (other.y == 0.0f ? 0.0f : other.y * f_other);
            const float inv = total == 0.0f ? 0.0f : 1.0f / total;
            if ((warp & 3u) * 32 < m_rows) {
                const unsigned flat = flat0 + min(row, m_rows - 1), node = flat / a.group, head = last->kv_head * a.group + flat % a.group;
                T* out = static_cast<T*>(a.out) + static_cast<size_t>(last->row0 + node) * a.out_stride + static_cast<size_t>(head) * HD;
                float* po = a.part_o + piece_at(blockIdx.x * 2 + last->piece(), HD, 0, row);
                const unsigned c0 = w * (HD / 2);
#pragma unroll 1
                for (unsigned c = c0; c < c0 + HD / 2; c += 16) {
                    uint32_t x[16], y[16];
                    tc_ld16(o_at + w * HD + c, x);
                    tc_ld16(o_at + (w ^ 1u) * HD + c, y);
                    tc_wait_ld16(x, y);
                    float o[16];
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        o[i] = fmaf(last_l == 0.0f ? 0.0f : __uint_as_float(x[i]), f_own, other.y == 0.0f ? 0.0f : __uint_as_float(y[i]) * f_other);
                    if (row < m_rows) {
                        if (whole) {
                            uint32_t h[8];
#pragma unroll
                            for (int k = 0; k < 8; k++) h[k] = pack2<T>(o[2 * k] * inv, o[2 * k + 1] * inv);
                            st_row16(out + c, h, a.out_vec32);
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; i++) po[static_cast<size_t>(c + i) * kTcRows] = o[i];
                        }
                    }
                }
                if (row < m_rows) {
                    if (!whole && w == 0) a.part_ml[(blockIdx.x * 2 + last->piece()) * kTcRows + row] = make_float2(top, total);
                    if (fix && total != 0.0f) add_bad_values<T, HD>(a, last, node, head, ref, total, out, whole ? nullptr : po, c0, c0 + HD / 2);
                }
            }
            tc_fence_before();
            meet(1);  // the accumulators may be written again
            pending = false;
        };
        float m = 0.0f, l = 0.0f;  // of the block, for this stream
        bool begun = false;        // a tile of this stream has gone into the accumulator
        // Scores that the row must not see become -inf, where they lie; 32 at a time, and only where some row of the warp has any.
        const auto hide = [&](uint32_t s_at, unsigned seen) {
            if (!__any_sync(0xffffffffu, seen != 0xffffffffu)) return;
            uint32_t x[32];
            tc_ld32(s_at, x);
            tc_wait_ld(x);
#pragma unroll
            for (int c = 0; c < 32; c++) x[c] = (seen >> c) & 1u ? x[c] : 0xff800000u;
            tc_st32(s_at, x);
        };
        // A row's 128 scores to weights, in two passes of 32 at a time with the next 32 on their way: the maximum, then the
        // weights.
        const auto weigh = [&](uint32_t s_at, unsigned i) {
            uint32_t v[2][32];
            float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            tc_ld32(s_at, v[0]);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                uint32_t(&x)[32] = v[j & 1];
                tc_wait_ld(x);
                tc_ld32(s_at + 32 * ((j + 1) & 3), v[(j + 1) & 1]);  // after the last, the first again
#pragma unroll
                for (int c = 0; c < 32; c += 8) {
#pragma unroll
                    for (int k = 0; k < 4; k++) tops[k] = fmaxf(fmaxf(tops[k], __uint_as_float(x[c + k])), __uint_as_float(x[c + k + 4]));
                }
            }
            float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
            if (top != -INFINITY) top *= scale;
            if (__any_sync(0xffffffffu, top > m + Weights<T>::kLag)) {
                const float before = m;
                if (top > m + Weights<T>::kLag) m = top;
                const float f = before == -INFINITY ? 0.0f : ex2(before - m);
                l *= f;
                if (begun) {
                    // the stream's earlier product has to be in the accumulator
                    const unsigned earlier = t + i - 2;
                    ok = __all_sync(0xffffffffu, tc_wait(sfree(earlier % S::kScores), (earlier / S::kScores) & 1u, a.wait_limit, gave_up));
                    tc_fence_after();
                    for (int c = 0; c < HD / 32; c++) {
                        uint32_t o[32];
                        tc_ld32(o_at + w * HD + 32 * c, o);
                        tc_wait_ld(o);
#pragma unroll
                        for (int k = 0; k < 32; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                        tc_st32(o_at + w * HD + 32 * c, o);
                    }
                }
            }
            const float ref = (m == -INFINITY ? 0.0f : m) - Weights<T>::kUp;
            const float2 scale2 = make_float2(scale, scale), ref2 = make_float2(-ref, -ref);
            float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                uint32_t(&x)[32] = v[j & 1];
                tc_wait_ld(x);
                if (j < 3) tc_ld32(s_at + 32 * (j + 1), v[(j + 1) & 1]);
                uint32_t p[16];
#pragma unroll
                for (int c = 0; c < 16; c++) {
                    float2 z = fma2(make_float2(__uint_as_float(x[2 * c]), __uint_as_float(x[2 * c + 1])), scale2, ref2);
                    z.x = ex2(z.x);
                    z.y = ex2(z.y);
                    sum[c & 1] = add2(sum[c & 1], z);
                    p[c] = pack2<T>(z.x, z.y);
                }
                tc_st16(s_at + 16 * j, p);
            }
            l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            tc_wait_st();
        };
        // V rows behind the last position are cleared (they may hold anything, and 0 * NaN is NaN); infinities and NaNs of
        // drafted ones become 0, as rows that do not see them must not get them: add_bad_values.
        // `helpers` threads, this one number `me` of them, share it: the warps that have no rows, or all four.
        const auto clear_v = [&](unsigned i, unsigned n, int valid, int drafted, unsigned me, unsigned helpers) {
            const unsigned at = 2 * (FEW ? ring_t : t) + v_place<HD>(i, n), slot = at % S::kSlots;
            ok = __all_sync(0xffffffffu, ok && tc_wait(full(slot), (at / S::kSlots) & 1u, a.wait_limit, gave_up));
            if (!ok) return;
            unsigned char* v_at = tc_smem + S::kRing + slot * S::kTile;
            const unsigned pieces = S::kSubs * 8;  // of 16 bytes, to a row
            for (unsigned e = me; e < (kTcKeys - valid) * pieces; e += helpers) {
                const unsigned r = valid + e / pieces, c = e % pieces;
                *reinterpret_cast<uint4*>(v_at + (c / 8) * S::kPanel + r * 128 + (c % 8) * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            // eight threads to a panel row
            const unsigned g8 = me >> 3, c8 = me & 7u;
            for (int r = drafted + static_cast<int>(g8); r < valid; r += static_cast<int>(helpers >> 3)) {
#pragma unroll
                for (int c = 0; c < S::kSubs; c++) {
                    if (make_finite<T>(reinterpret_cast<uint4*>(v_at + c * S::kPanel + r * 128 + c8 * 16))) misc[2 + (units & 3u)] = 1;
                }
            }
            proxy_fence();
        };
        bool few = false;  // the block before was one of few rows
        if (place.seq >= a.n_seqs) ok = false;
        while (ok) {
            ok = __all_sync(0xffffffffu, tc_wait(ufull + 8 * (units % S::kUnits), (units / S::kUnits) & 1u, a.wait_limit, gave_up));
            if (!ok) break;
            const TcUnit* now = described + units % S::kUnits;
            const unsigned n = now->n;
            if (n == 0 && !pending) break;
            const unsigned flat0 = now->block() * a.block_rows, m_rows = rows_of(a, now->drafted, now->block());
            if (FEW && n && m_rows <= kFewRows) {
                if (pending) finish();
                ok = few_rows<T, HD>(a, now, units, ring_t, met, ok);
                met ^= 1u;  // they met three times
                few = true;
                ring_t += n;
                units++;
                continue;
            }
            if (FEW && few && n) meet(0);  // what the block before left in shared memory has been read
            few = false;
            const unsigned node = (flat0 + min(row, m_rows - 1)) / a.group;
            const int pos_first = static_cast<int>(now->k0) * kTcKeys, ctx = now->ctx();
            const bool busy = (warp & 3u) * 32 < m_rows;  // some row of the warp is there
            // the row's mask is asked for now and needed with the last tiles
            unsigned long long w0 = 0, w1 = 0;
            if (n && a.mask && pos_first + static_cast<int>(n) * kTcKeys > ctx) {
                const unsigned long long* mask = a.mask + static_cast<size_t>(now->row0 + node) * a.mask_words;
                w0 = mask[0];
                if (a.mask_words > 1) w1 = mask[1];
            }
            m = -INFINITY;
            l = 0.0f;
            begun = false;
            unsigned i = (t ^ w) & 1u;
            do {
                const unsigned b = (t + i) % S::kScores;
                bool has = ok && i < n;
                if (has) ok = has = __all_sync(0xffffffffu, tc_wait(sfull(b), ((t + i) / S::kScores) & 1u, a.wait_limit, gave_up));
                if (has) {
                    tc_fence_after();
                    const int pos0 = pos_first + static_cast<int>(i) * kTcKeys;
                    const uint32_t s_at = tmem + b * 128 + lanes;
                    const bool masked = pos0 + kTcKeys > ctx;  // drafted rows, or the end, are in the tile
                    const int len = static_cast<int>(now->len);
                    if (busy) {
                        if (masked) {
                            const TreeSeq seq{now->row0, now->drafted, ctx, len, 0u};
#pragma unroll 1
                            for (int j = 0; j < 4; j++)
                                hide(s_at + 32 * j, seq.n <= 128 ? tree_visible2(a, seq, node, pos0 + 32 * j, w0, w1) : tree_visible(a, seq, node, pos0 + 32 * j));
                            tc_wait_st();
                        }
                        weigh(s_at, i);
                    }
                    if (masked) {
                        const unsigned first = min((m_rows + 31) / 32, 4u) & 3u;  // warps 0 .. first - 1 have rows, unless all do
                        if ((warp & 3u) >= first) clear_v(i, n, min(kTcKeys, len - pos0), max(0, ctx - pos0), row - first * 32, 128 - first * 32);
                    }
                    begun = true;
                }
                if (pending) finish();  // its last product ran while this tile's weights were worked out
                if (has) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(pready(b));
                }
                i += 2;
            } while (i < n);
            if (n == 0) break;
            last_m = m;
            last_l = l;
            pending = true;
            t += n;
            ring_t += n;
            units++;
            big_units++;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (tid == 0 && *gave_up) atomicOr(a.err_word, kErrTimeout);
    if (warp == 8) tc_dealloc(tmem, 512);
}

// Joins the pieces of blocks that several CTAs share. CTA c stands at the border between shares c and c + 1; the CTAs at
// the borders inside one block (eight CTAs to a border) divide it among them in parts of 8 rows by 32 columns, a thread to a
// value, or, of more than eight pieces, 8 rows by 8 columns, four threads to a value with a quarter of the pieces each.
// Eight pieces are in flight at a time. (Always by quarters, blocks of few pieces took 12 us longer over 128-row chunks;
// never, one block in 148 pieces took 25 us longer.) The walk to the block is done while the
// attention kernel still runs: what it reads was there before that kernel began.
template <typename T>
__global__ void __launch_bounds__(256) tree_join_tc_kernel(const TreeArgs a, unsigned shares) {
    pdl_launch();
    __shared__ unsigned long long sh[2 * 8 + 4];
    __shared__ float weight[kMaxShares + 1][8];
    __shared__ float row_sum[8];
    __shared__ float quarter[3][64];
    const unsigned c = blockIdx.x + 1;
    const TreePlace p = tree_locate<kTcKeys, 256>(a, sh, false, [&](unsigned total) {
        const TreeShares s(total, shares);
        return c < s.g ? s.first(c) : total;
    });
    if (p.seq >= a.n_seqs) {
        pdl_wait();
        return;
    }
    const TreeShares s(p.total, shares);
    const unsigned border = s.first(c);
    const TreeSeq q = tree_seq(a, p.seq, false);
    const unsigned kt = (static_cast<unsigned>(q.len) + kTcKeys - 1) / kTcKeys;
    const unsigned rows_all = q.n * a.group, blocks = (rows_all + a.block_rows - 1) / a.block_rows;
    const unsigned unit = (border - p.base) / kt;
    const unsigned t0 = p.base + unit * kt;
    const unsigned first = s.owner(t0) + 1, last = s.owner(t0 + kt - 1);  // borders inside the block
    const unsigned n_borders = last - first + 1, n_pieces = n_borders + 1;
    const unsigned kv_head = unit / blocks, block = unit - kv_head * blocks;
    const unsigned m_rows = min(a.block_rows, rows_all - block * a.block_rows);
    const unsigned slices = n_pieces > 8 ? 4u : 1u, part_cols = 32 / slices;
    const unsigned cols = a.head_dim / part_cols, parts = (m_rows + 7) / 8 * cols;
    const unsigned mine = (c - first) * gridDim.y + blockIdx.y, of = n_borders * gridDim.y;
    const unsigned part0 = parts * mine / of, part1 = parts * (mine + 1) / of;
    pdl_wait();
    if (border == t0) return;
    // piece x (0 ..) is left by share first - 1 + x; only the first of them may be a CTA's second block
    const bool second = s.first(first - 1) < t0;
    const auto piece = [&](unsigned x) { return (first - 1 + x) * 2 + (x == 0 && second ? 1u : 0u); };
    const unsigned r = threadIdx.x & 7u, in_part = (threadIdx.x >> 3) % part_cols, slice = threadIdx.x / (8 * part_cols), lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    unsigned rows_at = 0xffffffffu;
    for (unsigned part = part0; part < part1; part++) {
        const unsigned row0 = part / cols * 8, col = part % cols * part_cols + in_part;
        if (slices > 1 || row0 != rows_at) __syncthreads();  // what the part before left in shared memory has been read
        if (row0 != rows_at) {
            // a warp takes a row: the largest maximum, then the weights and their sum
            rows_at = row0;
            const bool in = row0 + warp < m_rows;
            float top = -INFINITY, l = 0.0f;
            if (in)
                for (unsigned x = lane; x < n_pieces; x += 32) top = fmaxf(top, a.part_ml[static_cast<size_t>(piece(x)) * kTcRows + row0 + warp].x);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            for (unsigned x = lane; x < n_pieces; x += 32) {
                float w = 0.0f;  // stays 0 where nothing of a piece was visible
                if (in) {
                    const float2 ml = a.part_ml[static_cast<size_t>(piece(x)) * kTcRows + row0 + warp];
                    if (ml.y != 0.0f) {
                        w = ex2(ml.x - (top == -INFINITY ? 0.0f : top));
                        l = fmaf(ml.y, w, l);
                    }
                }
                weight[x][warp] = w;
            }
            l = warp_sum(l);
            if (lane == 0) row_sum[warp] = l;
            __syncthreads();
        }
        const unsigned row = row0 + r;
        float acc = 0.0f;
        if (row < m_rows) {
            const unsigned x1 = n_pieces * (slice + 1) / slices;
#pragma unroll 8
            for (unsigned x = n_pieces * slice / slices; x < x1; x++) {
                const float w = weight[x][r], o = a.part_o[piece_at(piece(x), a.head_dim, col, row)];
                acc = w == 0.0f ? acc : fmaf(o, w, acc);
            }
        }
        if (slices > 1) {
            if (slice) quarter[slice - 1][threadIdx.x & 63u] = acc;
            __syncthreads();
            if (slice == 0) acc = ((acc + quarter[0][threadIdx.x]) + quarter[1][threadIdx.x]) + quarter[2][threadIdx.x];
        }
        if (slice || row >= m_rows) continue;
        const unsigned flat = block * a.block_rows + row, node = flat / a.group, head = kv_head * a.group + flat % a.group;
        const float l = row_sum[r];
        static_cast<T*>(a.out)[static_cast<size_t>(q.row0 + node) * a.out_stride + static_cast<size_t>(head) * a.head_dim + col] = from_f32<T>(l == 0.0f ? 0.0f : acc / l);
    }
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

// q as [row][query head][column], fetched as the rows of a block: the heads of one key head by 128 / group drafted rows.
// What a box holds of another sequence's rows is computed and thrown away; behind the last row there are zeros.
bool encode_q(CUtensorMap* map, const TreeArgs& a, bool half) {
    const EncodeTiled enc = encode_tiled();
    if (!enc) return false;
    const cuuint64_t dims[3] = {a.head_dim, a.n_q_heads, a.rows};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(a.head_dim) * 2, a.q_stride * 2};
    const cuuint32_t box[3] = {64, a.group, kTcRows / a.group}, step[3] = {1, 1, 1};
    return enc(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(a.q), dims, strides, box, step,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

unsigned tc_shares(const lokal_cuda_ctx* ctx) { return static_cast<unsigned>(ctx->sm_count) < kMaxShares ? static_cast<unsigned>(ctx->sm_count) : kMaxShares; }

template <typename T, int HD>
int launch_tc(lokal_cuda_ctx* ctx, cudaStream_t s, const TreeArgs& a) {
    CUtensorMap map_q, map_k, map_v;
    constexpr bool half = std::is_same<T, __half>::value;
    if (!encode_q(&map_q, a, half) || !encode_store(&map_k, a, a.k, half) || !encode_store(&map_v, a, a.v, half))
        return ctx->fail(LOKAL_ERR_CUDA, "tree_attn: q or a store cannot be described to the copy engine");
    const unsigned shares = tc_shares(ctx);
    // Few rows on average: the kernel that looks at each block (figures at the top).
    if (HD == 64 && static_cast<unsigned long long>(a.rows) * a.group <= static_cast<unsigned long long>(a.n_seqs) * kFewRows)
        launch_staged(tree_attn_tc_kernel<T, HD, HD == 64>, shares, kTcThreads, TcShape<HD>::kBytes, s, a, map_q, map_k, map_v);
    else
        launch_staged(tree_attn_tc_kernel<T, HD, false>, shares, kTcThreads, TcShape<HD>::kBytes, s, a, map_q, map_k, map_v);
    LOKAL_CHECK_LAUNCH(ctx, "tree_attn_tc_kernel");
    launch_k(tree_join_tc_kernel<T>, dim3(shares - 1, 8), 256, 0, s, a, shares);
    LOKAL_CHECK_LAUNCH(ctx, "tree_join_tc_kernel");
    return LOKAL_OK;
}

}  // namespace

unsigned tree_tc_block(const TreeArgs& a) { return kTcRows / a.group * a.group; }

size_t tree_tc_rows(const lokal_cuda_ctx* ctx) { return static_cast<size_t>(tc_shares(ctx)) * 2 * kTcRows; }

// Rows the copy engine can take (16-byte grid), and a scale that leaves a maximum a maximum and -inf what it is.
bool tree_tc_takes(const TreeArgs& a, int dtype, int kv_dtype) {
    return dtype == kv_dtype && dtype != LOKAL_F32 && (a.head_dim == 64 || a.head_dim == 128) && a.group <= kTcRows && a.scale_log2 > 0.0f && a.row_bytes % 16 == 0 && aligned_to(a.k, 16) &&
           aligned_to(a.v, 16) && aligned_to(a.q, 16) && aligned_to(a.out, 16) && a.q_stride % 8 == 0 && a.out_stride % 8 == 0;
}

int launch_tree_tc(lokal_cuda_ctx* ctx, cudaStream_t s, const TreeArgs& a, int dtype) {
    if (dtype == LOKAL_F16) return a.head_dim == 64 ? launch_tc<__half, 64>(ctx, s, a) : launch_tc<__half, 128>(ctx, s, a);
    return a.head_dim == 64 ? launch_tc<__nv_bfloat16, 64>(ctx, s, a) : launch_tc<__nv_bfloat16, 128>(ctx, s, a);
}

}  // namespace lokal
