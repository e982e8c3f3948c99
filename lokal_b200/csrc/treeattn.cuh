// What the three attention kernels (treeattn_tc.cu: 16-bit rows; treeattn_mma.cu: f32 accuracy; treeattn.cu: the rest) and
// the launch that joins their pieces share: the arguments, the walk over the work, the visibility of drafted rows.
//
// The work of a call is a list of tiles: for every sequence, key head and block of up to R query rows (a row is one drafted
// row and one of the query heads that share the key head), the sequence's keys in tiles of KT. The lengths are on the
// device, so the list is too: every CTA sums it up for itself and takes an equal, contiguous share of it, whatever the
// lengths. A block whose tiles fall to several CTAs is left by each as a piece (sums that are not yet divided, with
// their maximum) in the workspace, and tree_join_kernel puts the pieces together in the order of the keys: the result
// does not depend on timing.
#pragma once

#include "kvpool.cuh"

namespace lokal {

struct TreeArgs {
    const void* q;
    void* out;
    const char* k;  // base of the K store and of the V store
    const char* v;
    const uint32_t* slots;
    const int32_t* q_start;
    const unsigned long long* mask;  // NULL: a chain
    const int32_t* table;
    const int32_t* lens;
    unsigned* err_word;
    float* part_o;    // [CTA][2][R][head_dim] (tensor-core kernel: [CTA][2][head_dim][R])
    float2* part_ml;  // [CTA][2][R]: maximum (in units of log 2) and sum
    unsigned long long q_stride, out_stride, row_bytes;
    unsigned n_seqs, rows, mask_words, n_q_heads, n_kv_heads, group, head_dim;
    unsigned page_rows, page_shift, n_pages, n_slots, max_pages;
    unsigned block_rows;  // query rows of a block: at most R
    unsigned wait_limit, extra_tx;  // polls before a wait gives up; bytes announced that do not come (for the test of that)
    int out_vec32;        // rows of out start on 32-byte boundaries
    float scale_log2;  // scale * log2(e): the exponentials are powers of two
};

struct TreeSeq {
    unsigned row0, n;  // drafted rows row0 .. row0 + n
    int ctx, len;      // committed keys, all keys
    unsigned slot;
};

// A sequence the call cannot serve (its rows beyond the call's, more of them than the slot holds positions, a slot out
// of range) has n == 0: no row of it is read or written.
__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs& a, unsigned i, bool report) {
    const int s = a.q_start[i], e = a.q_start[i + 1];
    TreeSeq q{0u, 0u, 0, 0, a.slots ? a.slots[i] : i};
    bool ok = s >= 0 && e >= s && static_cast<unsigned>(e) <= a.rows && q.slot < a.n_slots;
    if (ok && e > s) {
        const int len = a.lens[q.slot];
        ok = len >= e - s && static_cast<unsigned>(len) <= a.max_pages << a.page_shift;
        if (ok) {
            q.row0 = static_cast<unsigned>(s);
            q.n = static_cast<unsigned>(e - s);
            q.len = len;
            q.ctx = len - (e - s);
        }
    }
    if (!ok && report) atomicOr(a.err_word, kErrPageRange);
    return q;
}

template <int KT>
__device__ __forceinline__ unsigned long long tree_tiles(const TreeArgs& a, const TreeSeq& q) {
    const unsigned long long blocks = (q.n * a.group + a.block_rows - 1) / a.block_rows;  // rows * heads fit 31 bits
    return blocks * a.n_kv_heads * ((static_cast<unsigned>(q.len) + KT - 1) / KT);
}

// The tiles of a call dealt to g CTAs: share c is [first(c), first(c + 1)), the first `extra` shares one tile longer.
struct TreeShares {
    unsigned g, len, extra;
    __device__ TreeShares(unsigned total, unsigned most) {
        g = total < most ? total : most;
        len = g ? total / g : 0u;
        extra = g ? total - len * g : 0u;
    }
    __device__ unsigned first(unsigned c) const { return c * len + min(c, extra); }
    __device__ unsigned owner(unsigned tile) const {
        const unsigned longer = extra * (len + 1);
        return tile < longer ? tile / (len + 1) : extra + (tile - longer) / len;
    }
};

struct TreePlace {
    unsigned total;  // tiles of the call
    unsigned base;   // tiles before sequence `seq`
    unsigned seq;    // n_seqs: nothing to do
};

// Whole CTA (NT threads): the sum of all tiles, then, for the tile number that `pick` makes of it, the sequence that
// holds the tile. `sh` is 2 * (NT / 32) + 4 words of shared memory. Sequences are summed NT at a time, so any number of
// them; up to NT take one trip to memory. More than 2^32 - 1 tiles are refused.
template <int KT, int NT, typename Pick>
__device__ TreePlace tree_locate(const TreeArgs& a, unsigned long long* sh, bool report, Pick pick) {
    constexpr unsigned kWarps = NT / 32;
    const unsigned lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    TreePlace p{0u, 0u, a.n_seqs};
    unsigned long long total = 0;
    if (a.n_seqs > NT) {
        unsigned long long sum = 0;
        for (unsigned i = threadIdx.x; i < a.n_seqs; i += NT) sum += tree_tiles<KT>(a, tree_seq(a, i, report));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) sh[warp] = sum;
        __syncthreads();
        for (unsigned w = 0; w < kWarps; w++) total += sh[w];
    }
    unsigned long long before = 0;
    for (unsigned base = 0; base < a.n_seqs; base += NT) {
        const unsigned i = base + threadIdx.x;
        const unsigned long long mine = i < a.n_seqs ? tree_tiles<KT>(a, tree_seq(a, i, report && a.n_seqs <= NT)) : 0;
        unsigned long long s = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long t = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= static_cast<unsigned>(o)) s += t;
        }
        __syncthreads();
        if (lane == 31) sh[kWarps + 2 + warp] = s;
        __syncthreads();
        unsigned long long off = before, all = 0;
        for (unsigned w = 0; w < kWarps; w++) {
            const unsigned long long t = sh[kWarps + 2 + w];
            if (w < warp) off += t;
            all += t;
        }
        if (a.n_seqs <= NT) total = all;
        if (total > 0xffffffffull) {
            if (report && threadIdx.x == 0) atomicOr(a.err_word, kErrPageRange);
            return p;
        }
        p.total = static_cast<unsigned>(total);
        const unsigned at = pick(p.total);
        if (at >= p.total) return p;
        if (at >= off + s - mine && at < off + s) {
            sh[kWarps] = off + s - mine;
            sh[kWarps + 1] = i;
        }
        before += all;
        if (at < before) break;  // the same for every thread
    }
    __syncthreads();
    if (p.total == 0) return p;
    p.base = static_cast<unsigned>(sh[kWarps]);
    p.seq = static_cast<unsigned>(sh[kWarps + 1]);
    return p;
}

// A block of rows of one sequence and key head, and the CTA's run of its key tiles.
struct TreeUnit {
    TreeSeq seq;
    unsigned kv_head, block;
    unsigned k0, k1;  // key tiles
    bool whole;       // all of the block's tiles: no piece is left
    unsigned piece;   // 0 if the block is the CTA's first, else 1
};

// Steps through the tiles [at, hi) of a CTA. Every role of a CTA walks for itself. `known` (shared memory, or NULL) holds
// the first kTreeKnown sequences of the walk: while the copies of K and V fill the memory's queues, a load takes four
// microseconds, and the two that a sequence needs depend on one another.
constexpr unsigned kTreeKnown = 30;  // what is left of a CTA's shared memory
template <int KT>
struct TreeWalk {
    unsigned at, hi, lo, base, cur_tiles, seq, first;
    const int4* known;
    TreeSeq cur;
    __device__ void start(const TreeArgs& a, const TreePlace& p, unsigned from, unsigned to, const int4* known_ = nullptr) {
        lo = at = from;
        hi = to;
        base = p.base;
        seq = first = p.seq;
        known = known_;
        cur = TreeSeq{0u, 0u, 0, 0, 0u};
        cur_tiles = 0;
        if (at < hi) load(a);
    }
    __device__ void load(const TreeArgs& a) {
        if (known && seq - first < kTreeKnown) {
            const int4 k = known[seq - first];
            cur = TreeSeq{static_cast<unsigned>(k.x), static_cast<unsigned>(k.y), k.z - k.y, k.z, static_cast<unsigned>(k.w)};
        } else {
            cur = tree_seq(a, seq, false);
        }
        cur_tiles = static_cast<unsigned>(tree_tiles<KT>(a, cur));
    }
    __device__ bool next(const TreeArgs& a, TreeUnit& u) {
        if (at >= hi) return false;
        while (at - base >= cur_tiles) {
            base += cur_tiles;
            seq++;
            if (seq >= a.n_seqs) return false;  // only if the arrays changed under the call
            load(a);
        }
        const unsigned off = at - base;
        const unsigned kt = (static_cast<unsigned>(cur.len) + KT - 1) / KT;
        const unsigned blocks = (cur.n * a.group + a.block_rows - 1) / a.block_rows;
        const unsigned unit = off / kt;
        u.seq = cur;
        u.kv_head = unit / blocks;
        u.block = unit - u.kv_head * blocks;
        u.k0 = off - unit * kt;
        u.k1 = min(kt, u.k0 + (hi - at));
        u.whole = u.k0 == 0 && u.k1 == kt;
        u.piece = lo >= base + unit * kt ? 0u : 1u;
        at += u.k1 - u.k0;
        return true;
    }
};

// 32 visibility bits of drafted row `node`: bit b is key position pos0 + b. Keys before ctx are committed and seen by
// all; u = position - ctx is the number of a drafted row.
__device__ __forceinline__ unsigned tree_visible(const TreeArgs& a, const TreeSeq& q, unsigned node, int pos0) {
    const int left = q.len - pos0;
    if (left <= 0) return 0u;
    unsigned in = left >= 32 ? 0xffffffffu : (1u << left) - 1u;
    const int u0 = pos0 - q.ctx;
    if (u0 + 31 < 0) return in;
    unsigned bits;
    if (!a.mask) {
        const int upto = static_cast<int>(node) - u0;  // drafted rows 0 .. node
        bits = upto >= 31 ? 0xffffffffu : upto < 0 ? 0u : (2u << upto) - 1u;
        return in & bits;
    }
    const unsigned long long* row = a.mask + static_cast<size_t>(q.row0 + node) * a.mask_words;
    if (u0 < 0) {
        const unsigned long long w = a.mask_words ? row[0] : 0ull;
        bits = (static_cast<unsigned>(w) << -u0) | ((1u << -u0) - 1u);
    } else {
        const unsigned word = static_cast<unsigned>(u0) >> 6, sh = static_cast<unsigned>(u0) & 63u;
        unsigned long long w = word < a.mask_words ? row[word] >> sh : 0ull;
        if (sh && word + 1 < a.mask_words) w |= row[word + 1] << (64u - sh);
        bits = static_cast<unsigned>(w);
    }
    return in & bits;
}

// The same 32 bits from the first two words of the row's mask, for sequences of up to 128 drafted rows.
__device__ __forceinline__ unsigned tree_visible2(const TreeArgs& a, const TreeSeq& q, unsigned node, int pos0, unsigned long long w0, unsigned long long w1) {
    if (!a.mask) return tree_visible(a, q, node, pos0);
    const int left = q.len - pos0, u0 = pos0 - q.ctx;
    if (left <= 0) return 0u;
    const unsigned in = left >= 32 ? 0xffffffffu : (1u << left) - 1u;
    if (u0 + 31 < 0) return in;
    if (u0 < 0) return in & ((static_cast<unsigned>(w0) << -u0) | ((1u << -u0) - 1u));
    const unsigned sh = static_cast<unsigned>(u0) & 63u;
    const unsigned long long lo = u0 < 64 ? w0 : u0 < 128 ? w1 : 0ull, hi = u0 < 64 ? w1 : 0ull;
    return in & static_cast<unsigned>((lo >> sh) | (sh ? hi << (64u - sh) : 0ull));
}

// Cache row of a position. A page that is not there is read as page 0 and reported: nothing outside the pool is touched.
__device__ __forceinline__ unsigned tree_page(const TreeArgs& a, unsigned slot, unsigned page_index) {
    const int page = a.table[static_cast<size_t>(slot) * a.max_pages + page_index];
    if (page < 0 || static_cast<unsigned>(page) >= a.n_pages) {
        atomicOr(a.err_word, kErrPageRange);
        return 0u;
    }
    return static_cast<unsigned>(page);
}

// launch_k for kernels whose tiles fill the shared memory of an SM: the whole of it is asked for.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_staged(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, Args&&... args) {
    {
        static std::mutex mu;
        static std::set<std::pair<int, const void*>> done;
        int dev = 0;
        cudaGetDevice(&dev);
        const std::pair<int, const void*> key(dev, reinterpret_cast<const void*>(kernel));
        std::lock_guard<std::mutex> g(mu);
        if (done.find(key) == done.end()) {
            cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
            if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
            if (e != cudaSuccess) return e;
            done.insert(key);
        }
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
}

// The tensor-core kernel (treeattn_tc.cu): whether it takes a call, the rows of its blocks and of the pieces it may leave,
// and its launch.
bool tree_tc_takes(const TreeArgs& a, int dtype, int kv_dtype);
unsigned tree_tc_block(const TreeArgs& a);
size_t tree_tc_rows(const lokal_cuda_ctx* ctx);
int launch_tree_tc(lokal_cuda_ctx* ctx, cudaStream_t s, const TreeArgs& a, int dtype);
// The kernel with f32 accuracy on the tensor cores (treeattn_mma.cu).
bool tree_mma_takes(const TreeArgs& a, int dtype, int kv_dtype);
size_t tree_mma_rows(const lokal_cuda_ctx* ctx, unsigned head_dim);
int launch_tree_mma(lokal_cuda_ctx* ctx, cudaStream_t s, const TreeArgs& a, int dtype, int kv_dtype);

// Joins the pieces of blocks that several CTAs share. CTA c stands at the border between shares c and c + 1; the CTAs at
// the borders inside one block divide its rows among them. A warp takes a row, or, where a CTA has fewer rows than warps,
// a part of a row's pieces (a single block may be in as many pieces as there are shares); 32 pieces are weighed at once,
// a lane each, and eight loads are in flight.
template <typename T, int R, int KT>
__global__ void __launch_bounds__(256) tree_join_kernel(const TreeArgs a, unsigned shares) {
    pdl_sync();
    __shared__ unsigned long long sh[2 * 8 + 4];
    __shared__ float part[8][256];
    __shared__ float part_l[8];
    const unsigned c = blockIdx.x + 1;
    const TreePlace p = tree_locate<KT, 256>(a, sh, false, [&](unsigned total) {
        const TreeShares s(total, shares);
        return c < s.g ? s.first(c) : total;
    });
    if (p.seq >= a.n_seqs) return;
    const TreeShares s(p.total, shares);
    const unsigned border = s.first(c);
    const TreeSeq q = tree_seq(a, p.seq, false);
    const unsigned kt = (static_cast<unsigned>(q.len) + KT - 1) / KT;
    const unsigned rows_all = q.n * a.group, blocks = (rows_all + a.block_rows - 1) / a.block_rows;
    const unsigned unit = (border - p.base) / kt;
    const unsigned t0 = p.base + unit * kt, t1 = t0 + kt;
    if (border == t0) return;
    const unsigned first = s.owner(t0) + 1, last = s.owner(t1 - 1);  // borders inside the block
    const unsigned n_borders = last - first + 1, n_pieces = n_borders + 1;
    const unsigned kv_head = unit / blocks, block = unit - kv_head * blocks;
    const unsigned m_rows = min(a.block_rows, rows_all - block * a.block_rows);
    const unsigned r0 = m_rows * (c - first) / n_borders, r1 = m_rows * (c - first + 1) / n_borders;
    const unsigned lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const bool first_is_0 = s.first(first - 1) >= t0;
    const unsigned rows = r1 - r0, parts = rows <= 1 ? 8u : rows <= 2 ? 4u : rows <= 4 ? 2u : 1u, step = 8u / parts;
    const unsigned x0 = n_pieces * (warp % parts) / parts, x1 = n_pieces * (warp % parts + 1) / parts;
    for (unsigned rr = r0; rr < r1; rr += step) {  // the same number of rounds for every warp
        const unsigned r = rr + warp / parts;
        const bool in = r < r1;
        // piece x (0 ..) is left by share first - 1 + x; only the first of them may be a CTA's second block
        auto slot_of = [&](unsigned x) {
            return (static_cast<size_t>(first - 1 + x) * 2 + (x == 0 && !first_is_0 ? 1 : 0)) * R + r;
        };
        float m = -INFINITY;
        if (in)
            for (unsigned x = lane; x < n_pieces; x += 32) m = fmaxf(m, a.part_ml[slot_of(x)].x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float ref = m == -INFINITY ? 0.0f : m;
        float acc[8];  // head_dim <= 256
#pragma unroll
        for (int j = 0; j < 8; j++) acc[j] = 0.0f;
        float l = 0.0f;
        for (unsigned x = in ? x0 : x1; x < x1; x += 32) {
            float w = 0.0f;  // stays 0 where nothing of a piece was visible
            if (x + lane < x1) {
                const float2 ml = a.part_ml[slot_of(x + lane)];
                if (ml.y != 0.0f) {
                    w = exp2f(ml.x - ref);
                    l = fmaf(ml.y, w, l);
                }
            }
            const unsigned n = min(32u, x1 - x);
#pragma unroll 8
            for (unsigned i = 0; i < n; i++) {
                const float wi = __shfl_sync(0xffffffffu, w, i);
                const float* o = a.part_o + slot_of(x + i) * a.head_dim;
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (j * 32 + lane < a.head_dim) acc[j] = wi == 0.0f ? acc[j] : fmaf(o[j * 32 + lane], wi, acc[j]);
            }
        }
        l = warp_sum(l);
        if (parts > 1) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < 8; j++) part[warp][j * 32 + lane] = acc[j];
            if (lane == 0) part_l[warp] = l;
            __syncthreads();
            if (warp % parts != 0) continue;
            for (unsigned y = 1; y < parts; y++) {
#pragma unroll
                for (int j = 0; j < 8; j++) acc[j] += part[warp + y][j * 32 + lane];
                l += part_l[warp + y];
            }
        }
        if (!in) continue;
        const unsigned flat = block * a.block_rows + r, node = flat / a.group, head = kv_head * a.group + flat % a.group;
        T* dst = static_cast<T*>(a.out) + static_cast<size_t>(q.row0 + node) * a.out_stride + static_cast<size_t>(head) * a.head_dim;
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (j * 32 + lane < a.head_dim) dst[j * 32 + lane] = from_f32<T>(l == 0.0f ? 0.0f : acc[j] / l);
    }
}

}  // namespace lokal
