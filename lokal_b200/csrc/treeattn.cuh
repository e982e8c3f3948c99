// What the two attention kernels (treeattn.cu: any type and shape; treeattn_tc.cu: 16-bit rows on the tensor cores) and
// the launch that joins their pieces share: the arguments, the walk over the work, the visibility of drafted rows.
//
// The work of a call is a list of tiles: for every sequence, key head and block of R query rows (a row is one drafted
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
    float* part_o;    // [CTA][2][R][head_dim]
    float2* part_ml;  // [CTA][2][R]: maximum (in units of log 2) and sum
    unsigned long long q_stride, out_stride, row_bytes;
    unsigned n_seqs, rows, mask_words, n_q_heads, n_kv_heads, group, head_dim;
    unsigned page_rows, page_shift, n_pages, n_slots, max_pages;
    unsigned wait_limit;
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

template <int R, int KT>
__device__ __forceinline__ unsigned long long tree_tiles(const TreeArgs& a, const TreeSeq& q) {
    const unsigned long long blocks = (static_cast<unsigned long long>(q.n) * a.group + R - 1) / R;
    return blocks * a.n_kv_heads * ((static_cast<unsigned>(q.len) + KT - 1) / KT);
}

// First tile of share c of g over `total` tiles.
__device__ __forceinline__ unsigned long long tree_share(unsigned long long total, unsigned c, unsigned g) {
    return total * c / g;
}

struct TreePlace {
    unsigned long long total;  // tiles of the call
    unsigned long long base;   // tiles before sequence `seq`
    unsigned seq;
};

// Whole CTA (NT threads): the sum of all tiles, then, for the tile number that `pick` makes of it, the sequence that
// holds the tile. `sh` is 2 * (NT / 32) + 4 words of shared memory. Sequences are summed NT at a time, so any number of them.
template <int R, int KT, int NT, typename Pick>
__device__ TreePlace tree_locate(const TreeArgs& a, unsigned long long* sh, bool report, Pick pick) {
    constexpr unsigned kWarps = NT / 32;
    const unsigned lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    unsigned long long sum = 0;
    for (unsigned i = threadIdx.x; i < a.n_seqs; i += NT) sum += tree_tiles<R, KT>(a, tree_seq(a, i, report));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sh[warp] = sum;
    __syncthreads();
    TreePlace p{0, 0, 0};
    for (unsigned w = 0; w < kWarps; w++) p.total += sh[w];
    const unsigned long long at = pick(p.total);
    if (at >= p.total) {
        p.seq = a.n_seqs;
        return p;
    }
    unsigned long long before = 0;
    for (unsigned base = 0; base < a.n_seqs; base += NT) {
        const unsigned i = base + threadIdx.x;
        const unsigned long long mine = i < a.n_seqs ? tree_tiles<R, KT>(a, tree_seq(a, i, false)) : 0;
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
        const unsigned long long from = off + s - mine;
        if (at >= from && at < off + s) {
            sh[kWarps] = from;
            sh[kWarps + 1] = i;
        }
        if (at < before + all) break;  // the same for every thread
        before += all;
    }
    __syncthreads();
    p.base = sh[kWarps];
    p.seq = static_cast<unsigned>(sh[kWarps + 1]);
    return p;
}

// A block of R rows of one sequence and key head, and the CTA's run of its key tiles.
struct TreeUnit {
    TreeSeq seq;
    unsigned kv_head, block;
    unsigned k0, k1;  // key tiles
    bool whole;       // all of the block's tiles: no piece is left
    unsigned piece;   // 0 if the block is the CTA's first, else 1
};

// Steps through the tiles [at, hi) of a CTA. Every role of a CTA walks for itself.
template <int R, int KT>
struct TreeWalk {
    unsigned long long at, hi, lo, base;
    unsigned seq;
    TreeSeq cur;
    unsigned long long cur_tiles;
    __device__ void start(const TreeArgs& a, const TreePlace& p, unsigned long long from, unsigned long long to) {
        lo = at = from;
        hi = to;
        base = p.base;
        seq = p.seq;
        cur = TreeSeq{0u, 0u, 0, 0, 0u};
        cur_tiles = 0;
        if (at < hi) load(a);
    }
    __device__ void load(const TreeArgs& a) {
        cur = tree_seq(a, seq, false);
        cur_tiles = tree_tiles<R, KT>(a, cur);
    }
    __device__ bool next(const TreeArgs& a, TreeUnit& u) {
        if (at >= hi) return false;
        while (at >= base + cur_tiles) {
            base += cur_tiles;
            seq++;
            if (seq >= a.n_seqs) return false;  // only if the arrays changed under the call
            load(a);
        }
        const unsigned long long off = at - base;
        const unsigned kt = (static_cast<unsigned>(cur.len) + KT - 1) / KT;
        const unsigned blocks = static_cast<unsigned>((static_cast<unsigned long long>(cur.n) * a.group + R - 1) / R);
        const unsigned long long unit = off / kt;
        u.seq = cur;
        u.kv_head = static_cast<unsigned>(unit / blocks);
        u.block = static_cast<unsigned>(unit % blocks);
        u.k0 = static_cast<unsigned>(off % kt);
        const unsigned long long left = hi - at;
        u.k1 = left < kt - u.k0 ? u.k0 + static_cast<unsigned>(left) : kt;
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

// The tensor-core kernel (treeattn_tc.cu): whether it takes a call, the rows of pieces it may leave, and its launch.
bool tree_tc_takes(const TreeArgs& a, int dtype, int kv_dtype);
size_t tree_tc_rows(const lokal_cuda_ctx* ctx);
int launch_tree_tc(lokal_cuda_ctx* ctx, cudaStream_t s, const TreeArgs& a, int dtype);

// Joins the pieces of blocks that several CTAs share. CTA c stands at the border between shares c and c + 1; the CTAs at
// the borders inside one block divide its rows among them. One warp per row.
template <typename T, int R, int KT>
__global__ void __launch_bounds__(256) tree_join_kernel(const TreeArgs a, unsigned shares) {
    pdl_sync();
    __shared__ unsigned long long sh[2 * 8 + 4];
    const unsigned c = blockIdx.x + 1;
    const TreePlace p = tree_locate<R, KT, 256>(a, sh, false, [&](unsigned long long total) {
        const unsigned g = total < shares ? static_cast<unsigned>(total) : shares;
        return c < g ? tree_share(total, c, g) : total;
    });
    if (p.seq >= a.n_seqs) return;
    const unsigned g = p.total < shares ? static_cast<unsigned>(p.total) : shares;
    const unsigned long long border = tree_share(p.total, c, g);
    const TreeSeq q = tree_seq(a, p.seq, false);
    const unsigned kt = (static_cast<unsigned>(q.len) + KT - 1) / KT;
    const unsigned rows_all = q.n * a.group, blocks = (rows_all + R - 1) / R;
    const unsigned long long unit = (border - p.base) / kt;
    const unsigned long long t0 = p.base + unit * kt, t1 = t0 + kt;
    if (border == t0) return;
    // borders inside (t0, t1): floor(total * x / g) > t0 and < t1
    const unsigned first = static_cast<unsigned>(((t0 + 1) * g + p.total - 1) / p.total);
    const unsigned last = static_cast<unsigned>((t1 * g + p.total - 1) / p.total) - 1u < g - 1u
                              ? static_cast<unsigned>((t1 * g + p.total - 1) / p.total) - 1u : g - 1u;
    const unsigned n_borders = last - first + 1;
    const unsigned kv_head = static_cast<unsigned>(unit / blocks), block = static_cast<unsigned>(unit % blocks);
    const unsigned m_rows = min(static_cast<unsigned>(R), rows_all - block * R);
    const unsigned r0 = m_rows * (c - first) / n_borders, r1 = m_rows * (c - first + 1) / n_borders;
    const unsigned lane = threadIdx.x & 31u;
    const bool first_is_0 = tree_share(p.total, first - 1, g) >= t0;
    for (unsigned r = r0 + (threadIdx.x >> 5); r < r1; r += 8) {
        const unsigned flat = block * R + r, node = flat / a.group, head = kv_head * a.group + flat % a.group;
        // piece x (0 ..) is left by share first - 1 + x; only the first of them may be a CTA's second block
        auto slot_of = [&](unsigned x) {
            return (static_cast<size_t>(first - 1 + x) * 2 + (x == 0 && !first_is_0 ? 1 : 0)) * R + r;
        };
        float m = -INFINITY;
        for (unsigned x = lane; x <= n_borders; x += 32) m = fmaxf(m, a.part_ml[slot_of(x)].x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float ref = m == -INFINITY ? 0.0f : m;
        float acc[8];  // head_dim <= 256
#pragma unroll
        for (int j = 0; j < 8; j++) acc[j] = 0.0f;
        float l = 0.0f;
        for (unsigned x = 0; x <= n_borders; x++) {
            const size_t s = slot_of(x);
            const float2 ml = a.part_ml[s];
            if (ml.y == 0.0f) continue;  // nothing of this piece was visible
            const float w = exp2f(ml.x - ref);
            l = fmaf(ml.y, w, l);
            const float* o = a.part_o + s * a.head_dim;
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (j * 32 + lane < a.head_dim) acc[j] = fmaf(o[j * 32 + lane], w, acc[j]);
        }
        T* dst = static_cast<T*>(a.out) + static_cast<size_t>(q.row0 + node) * a.out_stride + static_cast<size_t>(head) * a.head_dim;
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (j * 32 + lane < a.head_dim) dst[j * 32 + lane] = from_f32<T>(l == 0.0f ? 0.0f : acc[j] / l);
    }
}

}  // namespace lokal
