// A K/V cache in pages: which pages a sequence holds, and the copies that sharing, accepting and compacting need.
//
// The cache of a layer is one store for K and one for V, rows of `row_bytes`, addressed like the cache rows of
// kvstage.cu. Here the rows are grouped into pages of `page_rows`; page p is rows [p * page_rows, (p + 1) * page_rows)
// of EVERY store. Three integer arrays in device memory say who holds what:
//   table[slot][i]  page of positions [i * page_rows, (i + 1) * page_rows) of a slot, -1 where it holds none
//   lens[slot]      positions that the slot holds (pages 0 .. ceil(lens / page_rows) - 1 are there)
//   refs[page]      how many table entries name the page; 0 = free
// They stay on the device so that a decode loop (draft, verify, accept, grow) needs no host round trip and can be
// captured. The host-side twin of the reference is one linear region per slot (kvstage.cu); it has no pages.
//
// Every result is determined by the state before the call: new pages are the lowest-numbered free ones and are
// handed out in list order (prefix sums, never the order in which atomics arrive; the atomics on refs are integer
// adds, which commute). An entry that cannot be carried out is skipped and reported at the next synchronisation.
//
// Bound by memory: the integers are a few kilobytes, the rows are what costs. Calls that hand out pages (reserve, fork) and
// compact are two launches, a plan by one CTA and an apply over the whole GPU, joined by programmatic dependent launch; the
// others are one.
#include "common.cuh"
#include "kvpool.cuh"

#include <new>

namespace lokal {
namespace {

constexpr unsigned kPlanThreads = 1024;

// The pool's scratch (device ints): what a plan hands to the apply launch that follows it in the stream.
struct PoolWork {
    int* n_copies;   // copies in the list
    int* n_used;     // compact: used pages
    int* seqs_done;  // accept: sequences that are done; 0 between calls
    int* copy_src;   // [n_pages] page
    int* copy_dst;   // [n_pages] page
    int* copy_rows;  // [n_pages] rows of the page that are copied
    int* free_list;  // [n_pages] the lowest free pages, ascending
    int* remap;      // [n_pages] compact: new page of a page that moves
    int* claim;      // [n_slots] first list entry that names the slot as its target
    int* ent_new;    // [n_slots] per entry: its first place in free_list (accept: new length), -1 = skipped
    int* ent_len;    // [n_slots] per entry: positions of the slot before the call (fork: of the source; accept: pages it holds)
    int* ent_cow;    // [n_slots] per entry: page that is copied before the slot writes to it, -1 = none
    int* arrived;    // [n_slots] accept: CTAs of a sequence that are done; 0 between calls
};

__host__ __device__ inline PoolWork pool_work(int* w, unsigned n_pages, unsigned n_slots) {
    PoolWork p;
    p.n_copies = w;
    p.n_used = w + 1;
    p.seqs_done = w + 2;
    w += 4;
    p.copy_src = w;
    p.copy_dst = p.copy_src + n_pages;
    p.copy_rows = p.copy_dst + n_pages;
    p.free_list = p.copy_rows + n_pages;
    p.remap = p.free_list + n_pages;
    p.claim = p.remap + n_pages;
    p.ent_new = p.claim + n_slots;
    p.ent_len = p.ent_new + n_slots;
    p.ent_cow = p.ent_len + n_slots;
    p.arrived = p.ent_cow + n_slots;
    return p;
}
inline size_t pool_work_ints(unsigned n_pages, unsigned n_slots) { return 4 + 5 * static_cast<size_t>(n_pages) + 5 * static_cast<size_t>(n_slots); }

// Exclusive prefix sum over the CTA (kPlanThreads threads) of one value per thread; `total` for everybody.
template <typename N>
__device__ __forceinline__ N block_scan(N v, N& total, N* part /* 33 values of shared memory */) {
    const unsigned lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    N s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const N t = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= static_cast<unsigned>(o)) s += t;
    }
    __syncthreads();  // part may still be read by the call before
    if (lane == 31) part[warp] = s;
    __syncthreads();
    if (warp == 0) {
        N w = part[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const N t = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= static_cast<unsigned>(o)) w += t;
        }
        part[lane] = w;
        if (lane == 31) part[32] = w;
    }
    __syncthreads();
    total = part[32];
    return s - v + (warp ? part[warp - 1] : 0);
}

// The first `need` free pages, ascending, into work.free_list; returns how many there are (at most `need`).
__device__ int collect_free(const PoolArgs& a, const PoolWork& w, int need, int* part) {
    int have = 0;
    for (unsigned base = 0; base < a.n_pages && have < need; base += 4 * kPlanThreads) {
        const unsigned p0 = base + 4 * threadIdx.x;
        int is_free[4], n = 0, total;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            is_free[j] = p0 + j < a.n_pages && a.refs[p0 + j] == 0;
            n += is_free[j];
        }
        int at = have + block_scan(n, total, part);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (is_free[j]) {
                if (at < need) w.free_list[at] = static_cast<int>(p0 + j);
                at++;
            }
        }
        have += total;
    }
    __syncthreads();
    return have < need ? have : need;
}

__device__ __forceinline__ bool page_ok(const PoolArgs& a, int p) { return p >= 0 && static_cast<unsigned>(p) < a.n_pages; }
__device__ __forceinline__ int pages_of(const PoolArgs& a, int len) { return (len + static_cast<int>(a.page_rows) - 1) >> a.page_shift; }

struct ListArgs {
    const uint32_t* src;      // fork: sources
    const uint32_t* dst;      // the slots that change
    const int32_t* new_lens;  // reserve / truncate
    unsigned n;
};

// FORK: entry i makes slot dst[i] a copy of slot src[i]. Otherwise (reserve): slot dst[i] grows to new_lens[i].
template <bool FORK>
__global__ void __launch_bounds__(kPlanThreads) pool_plan_kernel(const PoolArgs a, const ListArgs l) {
    pdl_sync();
    __shared__ int part[33];
    __shared__ long long part64[33];
    const PoolWork w = pool_work(a.work, a.n_pages, a.n_slots);
    // a slot that is named twice belongs to the first entry that names it
    for (unsigned i = threadIdx.x; i < l.n; i += kPlanThreads)
        if (l.dst[i] < a.n_slots) w.claim[l.dst[i]] = 0x7fffffff;
    __syncthreads();
    for (unsigned i = threadIdx.x; i < l.n; i += kPlanThreads)
        if (l.dst[i] < a.n_slots) atomicMin(w.claim + l.dst[i], static_cast<int>(i));
    __syncthreads();
    const int cap = static_cast<int>(a.max_pages << a.page_shift);
    long long need_before = 0;  // a list may ask for more pages than 32 bits count
    unsigned err = 0;
    for (unsigned base = 0; base < l.n; base += kPlanThreads) {
        const unsigned i = base + threadIdx.x;
        int need = 0, len = 0, cow = -1;
        bool ok = false;
        if (i < l.n) {
            const unsigned d = l.dst[i];
            ok = d < a.n_slots && w.claim[d] == static_cast<int>(i);
            if (FORK) {
                const unsigned s = l.src[i];
                ok = ok && s < a.n_slots && s != d && a.lens[d] == 0;
                if (ok) {
                    len = a.lens[s];
                    ok = len >= 0 && len <= cap;
                }
                if (ok && (len & static_cast<int>(a.page_rows - 1))) {
                    cow = a.table[static_cast<size_t>(s) * a.max_pages + (len >> a.page_shift)];
                    ok = page_ok(a, cow);
                    need = ok ? 1 : 0;
                }
            } else {
                const int want = ok ? l.new_lens[i] : 0;
                ok = ok && want >= 0 && want <= cap;
                if (ok) {
                    len = a.lens[d];
                    ok = len >= 0 && len <= cap;
                }
                if (ok && want > len) {
                    need = pages_of(a, want) - pages_of(a, len);
                    if (len & static_cast<int>(a.page_rows - 1)) {
                        // the slot will write into its last page: one that others hold too is copied first
                        const int last = a.table[static_cast<size_t>(d) * a.max_pages + (len >> a.page_shift)];
                        ok = page_ok(a, last);
                        if (ok && a.refs[last] > 1) {
                            cow = last;
                            need++;
                        }
                    }
                }
            }
            if (!ok) {
                need = 0;
                err |= kErrPageRange;
            }
        }
        long long total;
        const long long before = need_before + block_scan(static_cast<long long>(need), total, part64);
        need_before += total;
        if (i < l.n) {
            w.ent_new[i] = !ok ? -1 : static_cast<int>(before < a.n_pages ? before : a.n_pages);
            w.ent_len[i] = len;
            w.ent_cow[i] = ok ? cow : -1;
        }
    }
    const int have = collect_free(a, w, static_cast<int>(need_before < a.n_pages ? need_before : a.n_pages), part);
    // copies, in list order; entries that need pages past the last free one are skipped
    int n_copies = 0;
    for (unsigned base = 0; base < l.n; base += kPlanThreads) {
        const unsigned i = base + threadIdx.x;
        int copies = 0;
        if (i < l.n && w.ent_new[i] >= 0) {
            const int cow = w.ent_cow[i], len = w.ent_len[i];
            int need = cow >= 0 ? 1 : 0;
            if (!FORK) {
                const int want = l.new_lens[i];
                if (want > len) need += pages_of(a, want) - pages_of(a, len);
            }
            if (need > 0 && w.ent_new[i] + need > have) {
                w.ent_new[i] = -1;
                err |= kErrNoPages;
            } else {
                copies = cow >= 0 ? 1 : 0;
            }
        }
        int total;
        const int at = n_copies + block_scan(copies, total, part);
        if (copies) {
            w.copy_src[at] = w.ent_cow[i];
            w.copy_dst[at] = w.free_list[w.ent_new[i]];
            w.copy_rows[at] = w.ent_len[i] & static_cast<int>(a.page_rows - 1);
        }
        n_copies += total;
    }
    if (threadIdx.x == 0) *w.n_copies = n_copies;
    if (err) atomicOr(a.err_word, err);
}

// Copies of the list, all stores: a CTA takes 16 KB of one page of one store at a time, four vectors per thread in flight.
template <typename V>
__device__ __forceinline__ void run_copies(const PoolArgs& a, const int* src_page, const int* dst_page, const int* rows, unsigned n_copies) {
    constexpr unsigned kUnroll = 4, kTile = 256 * kUnroll;
    const unsigned row_vecs = static_cast<unsigned>(a.row_bytes / sizeof(V));
    const unsigned page_vecs = row_vecs << a.page_shift;
    const unsigned tiles = (page_vecs + kTile - 1) / kTile;
    const unsigned long long items = static_cast<unsigned long long>(n_copies) * a.n_stores * tiles;
    for (unsigned long long it = blockIdx.x; it < items; it += gridDim.x) {
        const unsigned tile = static_cast<unsigned>(it % tiles);
        const unsigned long long rest = it / tiles;
        const unsigned store = static_cast<unsigned>(rest % a.n_stores), c = static_cast<unsigned>(rest / a.n_stores);
        const int sp = src_page[c], dp = dst_page[c];
        if (!page_ok(a, sp) || !page_ok(a, dp)) {
            if (threadIdx.x == 0) atomicOr(a.err_word, kErrPageRange);
            continue;
        }
        const unsigned vecs = rows ? static_cast<unsigned>(rows[c]) * row_vecs : page_vecs;
        V* base = static_cast<V*>(a.stores[store]);
        const V* src = base + static_cast<size_t>(sp) * page_vecs;
        V* dst = base + static_cast<size_t>(dp) * page_vecs;
        V v[kUnroll];
        const unsigned e0 = tile * kTile + threadIdx.x;
#pragma unroll
        for (unsigned j = 0; j < kUnroll; j++)
            if (e0 + j * 256 < vecs) v[j] = src[e0 + j * 256];
#pragma unroll
        for (unsigned j = 0; j < kUnroll; j++)
            if (e0 + j * 256 < vecs) dst[e0 + j * 256] = v[j];
    }
}

template <bool FORK, typename V>
__global__ void __launch_bounds__(256) pool_apply_kernel(const PoolArgs a, const ListArgs l) {
    pdl_sync();
    const PoolWork w = pool_work(a.work, a.n_pages, a.n_slots);
    const unsigned stride = gridDim.x * 256, first = blockIdx.x * 256 + threadIdx.x;
    const unsigned long long cells = static_cast<unsigned long long>(l.n) * a.max_pages;
    for (unsigned long long c = first; c < cells; c += stride) {
        const unsigned i = static_cast<unsigned>(c / a.max_pages), p = static_cast<unsigned>(c % a.max_pages);
        const int at = w.ent_new[i];
        if (at < 0) continue;
        const int len = w.ent_len[i], cow = w.ent_cow[i];
        int32_t* row = a.table + static_cast<size_t>(l.dst[i]) * a.max_pages;
        if (FORK) {
            const int full = len >> a.page_shift;
            int page = -1;
            if (static_cast<int>(p) < full) {
                page = a.table[static_cast<size_t>(l.src[i]) * a.max_pages + p];
                if (page_ok(a, page)) atomicAdd(a.refs + page, 1);
                else atomicOr(a.err_word, kErrPageRange);
            } else if (static_cast<int>(p) == full && cow >= 0) {
                page = w.free_list[at];
                a.refs[page] = 1;
            }
            row[p] = page;
            if (p == 0) a.lens[l.dst[i]] = len;
        } else {
            const int want = l.new_lens[i];
            if (want <= len) continue;
            const int have = pages_of(a, len);
            if (static_cast<int>(p) >= have && static_cast<int>(p) < pages_of(a, want)) {
                const int page = w.free_list[at + (cow >= 0 ? 1 : 0) + static_cast<int>(p) - have];
                a.refs[page] = 1;
                row[p] = page;
            } else if (cow >= 0 && static_cast<int>(p) == have - 1) {
                const int page = w.free_list[at];
                a.refs[page] = 1;
                row[p] = page;
                atomicSub(a.refs + cow, 1);
            }
            if (p == 0) a.lens[l.dst[i]] = want;
        }
    }
    run_copies<V>(a, w.copy_src, w.copy_dst, w.copy_rows, static_cast<unsigned>(*w.n_copies));
}

// Page p of a slot is given back if no position below `want` lies in it. The table entry is taken out by an exchange, so
// that a slot which a list names twice gives every page back once.
__device__ __forceinline__ void give_back(const PoolArgs& a, unsigned slot, unsigned p, int want) {
    if (static_cast<long long>(p) << a.page_shift < want) return;
    const int old = atomicExch(a.table + static_cast<size_t>(slot) * a.max_pages + p, -1);
    if (page_ok(a, old)) atomicSub(a.refs + old, 1);
}

__global__ void __launch_bounds__(256) pool_truncate_kernel(const PoolArgs a, const ListArgs l) {
    pdl_sync();
    const unsigned i = blockIdx.y;
    const unsigned slot = l.dst[i];
    const int want = l.new_lens ? l.new_lens[i] : 0;
    if (slot >= a.n_slots || want < 0) {
        if (threadIdx.x == 0 && blockIdx.x == 0) atomicOr(a.err_word, kErrPageRange);
        return;
    }
    const unsigned p = blockIdx.x * 256 + threadIdx.x;
    if (p == 0) atomicMin(a.lens + slot, want);
    if (p < a.max_pages) give_back(a, slot, p, want);
}

// The k-th free page below n_used gets the k-th used page at or above n_used: as many of one as of the other, sources
// and targets apart, so the copies may run in any order.
__global__ void __launch_bounds__(kPlanThreads) pool_compact_plan_kernel(const PoolArgs a, int32_t* n_used_out) {
    pdl_sync();
    __shared__ int part[33];
    const PoolWork w = pool_work(a.work, a.n_pages, a.n_slots);
    int n = 0, used = 0;
    for (unsigned p = threadIdx.x; p < a.n_pages; p += kPlanThreads) n += a.refs[p] != 0;
    block_scan(n, used, part);
    int holes = 0, movers = 0;
    for (unsigned base = 0; base < a.n_pages; base += 4 * kPlanThreads) {
        const unsigned p0 = base + 4 * threadIdx.x;
        int hole[4], mover[4], nh = 0, nm = 0, total;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const unsigned p = p0 + j;
            const bool in = p < a.n_pages, is_used = in && a.refs[p] != 0, low = p < static_cast<unsigned>(used);
            hole[j] = in && low && !is_used;
            mover[j] = in && !low && is_used;
            nh += hole[j];
            nm += mover[j];
            if (in && !low) w.remap[p] = -1;
        }
        int h = holes + block_scan(nh, total, part);
        holes += total;
        int m = movers + block_scan(nm, total, part);
        movers += total;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (hole[j]) w.copy_dst[h++] = static_cast<int>(p0 + j);
            if (mover[j]) w.copy_src[m++] = static_cast<int>(p0 + j);
        }
    }
    __syncthreads();
    for (int c = static_cast<int>(threadIdx.x); c < movers; c += kPlanThreads) w.remap[w.copy_src[c]] = w.copy_dst[c];
    if (threadIdx.x == 0) {
        *w.n_copies = movers;
        *w.n_used = used;
        if (n_used_out) *n_used_out = used;
    }
}

template <typename V>
__global__ void __launch_bounds__(256) pool_compact_apply_kernel(const PoolArgs a) {
    pdl_sync();
    const PoolWork w = pool_work(a.work, a.n_pages, a.n_slots);
    const unsigned stride = gridDim.x * 256, first = blockIdx.x * 256 + threadIdx.x;
    const int n = *w.n_copies, used = *w.n_used;
    if (n == 0) return;
    for (unsigned c = first; c < static_cast<unsigned>(n); c += stride) {
        a.refs[w.copy_dst[c]] = a.refs[w.copy_src[c]];
        a.refs[w.copy_src[c]] = 0;
    }
    const unsigned long long cells = static_cast<unsigned long long>(a.n_slots) * a.max_pages;
    for (unsigned long long c = first; c < cells; c += stride) {
        const int page = a.table[c];
        if (page >= used && page_ok(a, page)) {
            const int to = w.remap[page];
            if (to >= 0) a.table[c] = to;
            else atomicOr(a.err_word, kErrPageRange);  // an entry that names a page nobody holds
        }
    }
    run_copies<V>(a, w.copy_src, w.copy_dst, nullptr, static_cast<unsigned>(n));
}

template <typename V>
__global__ void __launch_bounds__(256) pool_copy_kernel(const PoolArgs a, const int* src, const int* dst, unsigned n) {
    pdl_sync();
    run_copies<V>(a, src, dst, nullptr, n);
}

// ---- the accepted path of a drafted tree ----
struct AcceptArgs {
    const uint32_t* slots;
    const int32_t* q_start;
    const int32_t* accepted;  // [n_seqs][max_accept]
    const int32_t* counts;    // [n_seqs]
    unsigned n_seqs, max_accept;
};
constexpr unsigned kMaxAccept = 256;

// One thread per 16 bytes of a row of a store walks the path in order: rows c + a_0, c + a_1, ... move to c, c + 1, ...
// in place. The a_j ascend, so a_j >= j and a row is written only after every move that reads it: within a batch all
// loads come before the first store, and a later source lies behind every target so far. The row numbers of the path
// are worked out once per CTA.
//
// A row must not move into a page that another slot holds. Every CTA decides that, and the rest of what makes an entry
// good, for itself and from the state before the call: table, lengths and counts are changed by the last CTA of the
// launch, when all the others have read them. (Were a sequence cut as soon as it is done, a page that two sequences of the
// list share would be shared for some CTAs of the other and not for the rest.)
template <typename V>
__global__ void __launch_bounds__(256) pool_accept_kernel(const PoolArgs a, const AcceptArgs t) {
    pdl_sync();
    __shared__ int from[kMaxAccept], to[kMaxAccept];
    __shared__ int bad, held;
    const unsigned i = blockIdx.y;
    const unsigned slot = t.slots ? t.slots[i] : i;
    const PoolWork w = pool_work(a.work, a.n_pages, a.n_slots);
    if (threadIdx.x == 0) bad = held = 0;
    __syncthreads();
    const int drafts = t.q_start[i + 1] - t.q_start[i], count = t.counts[i];
    int len = 0, base = 0;
    bool ok = slot < a.n_slots && drafts >= 0 && count >= 0 && count <= drafts && count <= static_cast<int>(t.max_accept);
    if (ok) {
        len = a.lens[slot];
        base = len - drafts;
        ok = base >= 0 && len <= static_cast<int>(a.max_pages << a.page_shift);
    }
    const int32_t* row = a.table + static_cast<size_t>(ok ? slot : 0) * a.max_pages;
    if (ok) {
        const int32_t* acc = t.accepted + static_cast<size_t>(i) * t.max_accept;
        for (int j = static_cast<int>(threadIdx.x); j < count; j += 256) {
            const int x = acc[j];
            if (x < 0 || x >= drafts || (j > 0 && acc[j - 1] >= x)) {
                bad = 1;
                continue;
            }
            const int ps = row[(base + x) >> a.page_shift], pd = row[(base + j) >> a.page_shift];
            if (!page_ok(a, ps) || !page_ok(a, pd) || (x != j && a.refs[pd] > 1)) {
                bad = 1;
                continue;
            }
            const int m = static_cast<int>(a.page_rows) - 1;
            from[j] = (ps << a.page_shift) + ((base + x) & m);
            to[j] = (pd << a.page_shift) + ((base + j) & m);
        }
        // a slot that an earlier sequence of the list names too is that sequence's
        for (unsigned k = threadIdx.x; k < i; k += 256)
            if ((t.slots ? t.slots[k] : k) == slot) bad = 1;
    }
    __syncthreads();
    ok = ok && !bad;
    const int want = base + count;
    if (blockIdx.x == 0) {
        // what the cut behind the path needs to know: the new length, and how far the slot's pages go
        if (ok) {
            int end = 0;
            for (unsigned p = static_cast<unsigned>(pages_of(a, want)) + threadIdx.x; p < a.max_pages; p += 256)
                if (row[p] >= 0) end = static_cast<int>(p) + 1;
            if (end) atomicMax(&held, end);
        } else if (threadIdx.x == 0) {
            atomicOr(a.err_word, kErrPageRange);
        }
    }
    const unsigned row_vecs = static_cast<unsigned>(a.row_bytes / sizeof(V));
    const unsigned long long vecs = static_cast<unsigned long long>(row_vecs) * a.n_stores;
    for (unsigned long long e = static_cast<unsigned long long>(blockIdx.x) * 256 + threadIdx.x; ok && e < vecs; e += gridDim.x * 256ull) {
        V* base_v = static_cast<V*>(a.stores[e / row_vecs]) + e % row_vecs;
        constexpr int kBatch = 8;
        for (int j0 = 0; j0 < count; j0 += kBatch) {
            V v[kBatch];
#pragma unroll
            for (int j = 0; j < kBatch; j++)
                if (j0 + j < count) v[j] = base_v[static_cast<size_t>(from[j0 + j]) * row_vecs];
#pragma unroll
            for (int j = 0; j < kBatch; j++)
                if (j0 + j < count && from[j0 + j] != to[j0 + j]) base_v[static_cast<size_t>(to[j0 + j]) * row_vecs] = v[j];
        }
    }
    // The cuts behind the paths, by the launch's last CTA (in the one launch that the moves need; the counts are back at 0 for
    // the next call).
    __syncthreads();
    if (threadIdx.x == 0) {
        if (blockIdx.x == 0) {
            w.ent_new[i] = ok ? want : -1;
            w.ent_len[i] = held;
        }
        __threadfence();
        bad = atomicAdd(w.arrived + i, 1) == static_cast<int>(gridDim.x) - 1;
        if (bad) {
            w.arrived[i] = 0;
            __threadfence();
            bad = atomicAdd(w.seqs_done, 1) == static_cast<int>(gridDim.y) - 1;
            __threadfence();
        }
    }
    __syncthreads();
    if (!bad) return;
    if (threadIdx.x == 0) *w.seqs_done = 0;
    unsigned lanes = 32;  // to a sequence: a few pages are behind its path
    while (lanes > 1 && lanes * t.n_seqs > 256) lanes >>= 1;
    for (unsigned k = threadIdx.x / lanes; k < t.n_seqs; k += 256 / lanes) {
        const int cut = __ldcg(w.ent_new + k);
        const unsigned end = static_cast<unsigned>(__ldcg(w.ent_len + k)), of = t.slots ? t.slots[k] : k;
        if (cut < 0) continue;
        if (threadIdx.x % lanes == 0) a.lens[of] = cut;
        int32_t* pages = a.table + static_cast<size_t>(of) * a.max_pages;
        for (unsigned p0 = static_cast<unsigned>(pages_of(a, cut)) + threadIdx.x % lanes; p0 < end; p0 += 4 * lanes) {
            int old[4];
#pragma unroll
            for (unsigned j = 0; j < 4; j++) old[j] = p0 + j * lanes < end ? pages[p0 + j * lanes] : -1;
#pragma unroll
            for (unsigned j = 0; j < 4; j++) {
                if (p0 + j * lanes < end) pages[p0 + j * lanes] = -1;
                if (page_ok(a, old[j])) atomicSub(a.refs + old[j], 1);
            }
        }
    }
}

// ---- cache rows of token rows, the paged twin of kv_rows ----
struct PageRowsArgs {
    const int32_t* positions;
    long long pos0;
    const uint32_t* slots;
    unsigned slot0;
    unsigned long long rows;
    uint32_t* out;
};

__global__ void __launch_bounds__(256) pool_rows_kernel(const PoolArgs a, const PageRowsArgs r) {
    pdl_sync();
    const unsigned long long i = static_cast<unsigned long long>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= r.rows) return;
    const long long pos = r.positions ? static_cast<long long>(r.positions[i]) : r.pos0 + static_cast<long long>(i);
    const unsigned slot = r.slots ? r.slots[i] : r.slot0;
    unsigned out = LOKAL_KV_ROW_NONE;
    if (slot < a.n_slots && pos >= 0 && pos < a.lens[slot] && pos < static_cast<long long>(a.max_pages) << a.page_shift) {
        const int page = a.table[static_cast<size_t>(slot) * a.max_pages + (pos >> a.page_shift)];
        if (page_ok(a, page)) out = (static_cast<unsigned>(page) << a.page_shift) + (static_cast<unsigned>(pos) & (a.page_rows - 1));
    }
    if (out == LOKAL_KV_ROW_NONE) atomicOr(a.err_word, kErrPosRange);
    r.out[i] = out;
}

// Enough CTAs to have a few megabytes in flight, no more than there is work for.
unsigned copy_grid(const lokal_cuda_ctx* ctx, unsigned long long items) {
    const unsigned long long most = static_cast<unsigned long long>(ctx->sm_count) * 8;
    return static_cast<unsigned>(items < 1 ? 1 : items < most ? items : most);
}
unsigned long long copy_items(const lokal_kv_pool* p, unsigned long long copies) {
    const unsigned long long vecs = (p->a.row_bytes / (p->vec16 ? 16 : 2)) << p->a.page_shift;
    return copies * p->a.n_stores * ((vecs + 1023) / 1024);
}

// The pool as a launch of this context sees it: errors go to the context that makes the call.
PoolArgs args_of(const lokal_cuda_ctx* ctx, const lokal_kv_pool* p) {
    PoolArgs a = p->a;
    a.err_word = ctx->err_word;
    return a;
}

template <bool FORK>
int launch_plan_apply(lokal_cuda_ctx* ctx, cudaStream_t s, const lokal_kv_pool* p, const ListArgs& l, const char* what) {
    const PoolArgs a = args_of(ctx, p);
    launch_k(pool_plan_kernel<FORK>, 1, kPlanThreads, 0, s, a, l);
    LOKAL_CHECK_LAUNCH(ctx, what);
    // a copy per entry at most; the table cells are few against them
    const unsigned long long cells = (static_cast<unsigned long long>(l.n) * p->a.max_pages + 255) / 256;
    const unsigned long long items = copy_items(p, l.n);
    const unsigned grid = copy_grid(ctx, items > cells ? items : cells);
    if (p->vec16) launch_k(pool_apply_kernel<FORK, uint4>, grid, 256, 0, s, a, l);
    else launch_k(pool_apply_kernel<FORK, unsigned short>, grid, 256, 0, s, a, l);
    LOKAL_CHECK_LAUNCH(ctx, what);
    return LOKAL_OK;
}

int launch_truncate(lokal_cuda_ctx* ctx, cudaStream_t s, const lokal_kv_pool* p, const ListArgs& l) {
    launch_k(pool_truncate_kernel, dim3((p->a.max_pages + 255) / 256, l.n), 256, 0, s, args_of(ctx, p), l);
    LOKAL_CHECK_LAUNCH(ctx, "pool_truncate_kernel");
    return LOKAL_OK;
}

// Checks that every call on a pool makes of its list.
int check_list(lokal_cuda_ctx* ctx, const lokal_kv_pool* p, const char* what, size_t n, const void* a, const void* b, bool need_b) {
    if (n && (!a || (need_b && !b))) return ctx->fail(LOKAL_ERR_BAD_ARG, "%s: a list is null", what);
    if (!aligned_to(a, 4) || !aligned_to(b, 4)) return ctx->fail(LOKAL_ERR_MISALIGNED, "%s: a list is not 4-byte aligned", what);
    if (n > p->a.n_slots) return ctx->fail(LOKAL_ERR_BAD_ARG, "%s: %zu entries for a pool of %u slots", what, n, p->a.n_slots);
    if (n > 65535) return ctx->fail(LOKAL_ERR_BAD_ARG, "%s: more than 65535 entries in one call", what);
    return LOKAL_OK;
}

}  // namespace
}  // namespace lokal

#define LOKAL_POOL_ENTER(ctx, pool, what)                                                                       \
    if (!(ctx)) return LOKAL_ERR_BAD_ARG;                                                                       \
    lokal::DeviceGuard guard__((ctx)->device);                                                                  \
    if (!guard__.ok) return (ctx)->fail(LOKAL_ERR_CUDA, "cannot select device %d", (ctx)->device);              \
    if (!(pool)) return (ctx)->fail(LOKAL_ERR_BAD_ARG, what ": the pool is null");                              \
    if ((pool)->device != (ctx)->device)                                                                        \
    return (ctx)->fail(LOKAL_ERR_BAD_ARG, what ": the pool is on device %d, the context on %d", (pool)->device, (ctx)->device)

extern "C" {

int lokal_cuda_kv_pool_create(lokal_cuda_ctx* ctx, uint32_t page_rows, uint32_t n_pages, uint32_t n_slots, uint32_t max_pages,
                              int32_t* table, int32_t* lens, int32_t* refs, void* const* stores, uint32_t n_stores, size_t row_bytes,
                              lokal_kv_pool** out) {
    if (!ctx) return LOKAL_ERR_BAD_ARG;
    lokal::DeviceGuard guard(ctx->device);
    if (!guard.ok) return ctx->fail(LOKAL_ERR_CUDA, "cannot select device %d", ctx->device);
    if (!out) return ctx->fail(LOKAL_ERR_BAD_ARG, "kv_pool_create: output pointer is null");
    *out = nullptr;
    if (!table || !lens || !refs || !stores) return ctx->fail(LOKAL_ERR_BAD_ARG, "kv_pool_create: table, lens, refs and stores must be non-null");
    if (page_rows < 8 || page_rows > 256 || (page_rows & (page_rows - 1)))
        return ctx->fail(LOKAL_ERR_BAD_ARG, "kv_pool_create: page_rows %u is not a power of two from 8 to 256", page_rows);
    if (!n_pages || !n_slots || !max_pages || !n_stores) return ctx->fail(LOKAL_ERR_BAD_ARG, "kv_pool_create: pages, slots, table width and stores must be non-zero");
    if (static_cast<uint64_t>(n_pages) * page_rows > 0x7fffffffull || static_cast<uint64_t>(max_pages) * page_rows > 0x7fffff00ull)  // a key tile behind the last position still counts in 32 bits
        return ctx->fail(LOKAL_ERR_BAD_ARG, "kv_pool_create: more than 2^31 - 1 rows in a store or 2^31 - 256 positions in a slot");
    if (n_slots > 0x7fffffffu || n_stores > 65536) return ctx->fail(LOKAL_ERR_BAD_ARG, "kv_pool_create: too many slots or stores");
    if (row_bytes == 0 || row_bytes % 2 || row_bytes > (1u << 22)) return ctx->fail(LOKAL_ERR_BAD_ARG, "kv_pool_create: row_bytes %zu is zero, odd or above 4 MB", row_bytes);
    if (!lokal::aligned_to(table, 4) || !lokal::aligned_to(lens, 4) || !lokal::aligned_to(refs, 4))
        return ctx->fail(LOKAL_ERR_MISALIGNED, "kv_pool_create: an integer array is not 4-byte aligned");
    bool vec16 = row_bytes % 16 == 0;
    for (uint32_t i = 0; i < n_stores; i++) {
        if (!stores[i]) return ctx->fail(LOKAL_ERR_BAD_ARG, "kv_pool_create: store %u is null", i);
        if (!lokal::aligned_to(stores[i], 2)) return ctx->fail(LOKAL_ERR_MISALIGNED, "kv_pool_create: store %u is not aligned to its element size", i);
        vec16 = vec16 && lokal::aligned_to(stores[i], 16);
    }
    lokal_kv_pool* p = new (std::nothrow) lokal_kv_pool();
    if (!p) return ctx->fail(LOKAL_ERR_CUDA, "kv_pool_create: out of host memory");
    p->stores.reset(new (std::nothrow) void*[n_stores]);
    const size_t ints = lokal::pool_work_ints(n_pages, n_slots);
    void* dev = nullptr;
    cudaError_t e = p->stores ? cudaSuccess : cudaErrorMemoryAllocation;
    if (e == cudaSuccess) e = cudaMalloc(&dev, n_stores * sizeof(void*) + ints * sizeof(int));
    // waited for: a copy from pageable memory returns before it has arrived, and the streams of the calls to come do not
    // order themselves behind the default stream
    if (e == cudaSuccess) e = cudaMemsetAsync(dev, 0, n_stores * sizeof(void*) + ints * sizeof(int), ctx->host_stream);
    if (e == cudaSuccess) e = cudaMemcpyAsync(dev, stores, n_stores * sizeof(void*), cudaMemcpyHostToDevice, ctx->host_stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(ctx->host_stream);
    if (e != cudaSuccess) {
        if (dev) cudaFree(dev);
        delete p;
        cudaGetLastError();
        return ctx->fail(LOKAL_ERR_CUDA, "kv_pool_create: %s", cudaGetErrorString(e));
    }
    for (uint32_t i = 0; i < n_stores; i++) p->stores[i] = stores[i];
    unsigned shift = 0;
    while ((1u << shift) < page_rows) shift++;
    p->device = ctx->device;
    p->block = dev;
    p->vec16 = vec16;
    p->a = {table, lens, refs, static_cast<void**>(dev), reinterpret_cast<int*>(static_cast<void**>(dev) + n_stores), nullptr,
            page_rows, shift, n_pages, n_slots, max_pages, n_stores, row_bytes};
    *out = p;
    return LOKAL_OK;
}

int lokal_cuda_kv_pool_destroy(lokal_cuda_ctx* ctx, lokal_kv_pool* pool) {
    if (!ctx) return LOKAL_ERR_BAD_ARG;
    lokal::DeviceGuard guard(ctx->device);
    if (!guard.ok) return ctx->fail(LOKAL_ERR_CUDA, "cannot select device %d", ctx->device);
    if (!pool) return LOKAL_OK;
    const cudaError_t e = cudaFree(pool->block);
    delete pool;
    if (e != cudaSuccess) return ctx->fail(LOKAL_ERR_CUDA, "kv_pool_destroy: %s", cudaGetErrorString(e));
    return LOKAL_OK;
}

int lokal_cuda_kv_pool_reset(lokal_cuda_ctx* ctx, lokal_cuda_stream s, lokal_kv_pool* pool) {
    LOKAL_POOL_ENTER(ctx, pool, "kv_pool_reset");
    cudaStream_t st = static_cast<cudaStream_t>(s);
    const lokal::PoolArgs& a = pool->a;
    LOKAL_CUDA_TRY(ctx, cudaMemsetAsync(a.table, 0xff, static_cast<size_t>(a.n_slots) * a.max_pages * 4, st));
    LOKAL_CUDA_TRY(ctx, cudaMemsetAsync(a.lens, 0, static_cast<size_t>(a.n_slots) * 4, st));
    LOKAL_CUDA_TRY(ctx, cudaMemsetAsync(a.refs, 0, static_cast<size_t>(a.n_pages) * 4, st));
    return LOKAL_OK;
}

int lokal_cuda_kv_pool_rows(lokal_cuda_ctx* ctx, lokal_cuda_stream s, const lokal_kv_pool* pool, const int32_t* positions, int64_t pos0,
                            const uint32_t* slots, uint32_t slot0, size_t rows, uint32_t* rows_out) {
    LOKAL_POOL_ENTER(ctx, pool, "kv_pool_rows");
    if (!rows_out) return ctx->fail(LOKAL_ERR_BAD_ARG, "kv_pool_rows: output must be non-null");
    if (!positions && pos0 < 0) return ctx->fail(LOKAL_ERR_BAD_ARG, "kv_pool_rows: pos0 is negative");
    if (!lokal::aligned_to(rows_out, 4) || !lokal::aligned_to(positions, 4) || !lokal::aligned_to(slots, 4))
        return ctx->fail(LOKAL_ERR_MISALIGNED, "kv_pool_rows: a pointer is not 4-byte aligned");
    if (rows == 0) return LOKAL_OK;
    const unsigned long long blocks = (rows + 255) / 256;
    if (blocks > 0x7fffffffull) return ctx->fail(LOKAL_ERR_BAD_ARG, "kv_pool_rows: too many rows for one launch");
    lokal::PageRowsArgs r{positions, pos0, slots, slot0, rows, rows_out};
    lokal::launch_k(lokal::pool_rows_kernel, static_cast<unsigned>(blocks), 256, 0, static_cast<cudaStream_t>(s), lokal::args_of(ctx, pool), r);
    LOKAL_CHECK_LAUNCH(ctx, "pool_rows_kernel");
    return LOKAL_OK;
}

int lokal_cuda_kv_pool_reserve(lokal_cuda_ctx* ctx, lokal_cuda_stream s, lokal_kv_pool* pool, const uint32_t* slots,
                               const int32_t* new_lens, size_t n) {
    LOKAL_POOL_ENTER(ctx, pool, "kv_pool_reserve");
    int rc = lokal::check_list(ctx, pool, "kv_pool_reserve", n, slots, new_lens, true);
    if (rc != LOKAL_OK || n == 0) return rc;
    return lokal::launch_plan_apply<false>(ctx, static_cast<cudaStream_t>(s), pool, {nullptr, slots, new_lens, static_cast<unsigned>(n)}, "kv_pool_reserve");
}

int lokal_cuda_kv_pool_fork(lokal_cuda_ctx* ctx, lokal_cuda_stream s, lokal_kv_pool* pool, const uint32_t* src_slots,
                            const uint32_t* dst_slots, size_t n) {
    LOKAL_POOL_ENTER(ctx, pool, "kv_pool_fork");
    int rc = lokal::check_list(ctx, pool, "kv_pool_fork", n, src_slots, dst_slots, true);
    if (rc != LOKAL_OK || n == 0) return rc;
    return lokal::launch_plan_apply<true>(ctx, static_cast<cudaStream_t>(s), pool, {src_slots, dst_slots, nullptr, static_cast<unsigned>(n)}, "kv_pool_fork");
}

int lokal_cuda_kv_pool_truncate(lokal_cuda_ctx* ctx, lokal_cuda_stream s, lokal_kv_pool* pool, const uint32_t* slots,
                                const int32_t* new_lens, size_t n) {
    LOKAL_POOL_ENTER(ctx, pool, "kv_pool_truncate");
    int rc = lokal::check_list(ctx, pool, "kv_pool_truncate", n, slots, new_lens, false);
    if (rc != LOKAL_OK || n == 0) return rc;
    return lokal::launch_truncate(ctx, static_cast<cudaStream_t>(s), pool, {nullptr, slots, new_lens, static_cast<unsigned>(n)});
}

int lokal_cuda_kv_pool_compact(lokal_cuda_ctx* ctx, lokal_cuda_stream s, lokal_kv_pool* pool, int32_t* n_used) {
    LOKAL_POOL_ENTER(ctx, pool, "kv_pool_compact");
    if (!lokal::aligned_to(n_used, 4)) return ctx->fail(LOKAL_ERR_MISALIGNED, "kv_pool_compact: n_used is not 4-byte aligned");
    cudaStream_t st = static_cast<cudaStream_t>(s);
    lokal::launch_k(lokal::pool_compact_plan_kernel, 1, lokal::kPlanThreads, 0, st, lokal::args_of(ctx, pool), n_used);
    LOKAL_CHECK_LAUNCH(ctx, "pool_compact_plan_kernel");
    const unsigned long long cells = (static_cast<unsigned long long>(pool->a.n_slots) * pool->a.max_pages + 255) / 256;
    const unsigned long long items = lokal::copy_items(pool, (pool->a.n_pages + 1) / 2);
    const unsigned grid = lokal::copy_grid(ctx, items > cells ? items : cells);
    if (pool->vec16) lokal::launch_k(lokal::pool_compact_apply_kernel<uint4>, grid, 256, 0, st, lokal::args_of(ctx, pool));
    else lokal::launch_k(lokal::pool_compact_apply_kernel<unsigned short>, grid, 256, 0, st, lokal::args_of(ctx, pool));
    LOKAL_CHECK_LAUNCH(ctx, "pool_compact_apply_kernel");
    return LOKAL_OK;
}

int lokal_cuda_kv_pool_copy_pages(lokal_cuda_ctx* ctx, lokal_cuda_stream s, const lokal_kv_pool* pool, const int32_t* src_pages,
                                  const int32_t* dst_pages, size_t n) {
    LOKAL_POOL_ENTER(ctx, pool, "kv_pool_copy_pages");
    if (n && (!src_pages || !dst_pages)) return ctx->fail(LOKAL_ERR_BAD_ARG, "kv_pool_copy_pages: a list is null");
    if (!lokal::aligned_to(src_pages, 4) || !lokal::aligned_to(dst_pages, 4)) return ctx->fail(LOKAL_ERR_MISALIGNED, "kv_pool_copy_pages: a list is not 4-byte aligned");
    if (n > pool->a.n_pages) return ctx->fail(LOKAL_ERR_BAD_ARG, "kv_pool_copy_pages: %zu entries for a pool of %u pages", n, pool->a.n_pages);
    if (n == 0) return LOKAL_OK;
    const unsigned grid = lokal::copy_grid(ctx, lokal::copy_items(pool, n));
    cudaStream_t st = static_cast<cudaStream_t>(s);
    if (pool->vec16) lokal::launch_k(lokal::pool_copy_kernel<uint4>, grid, 256, 0, st, lokal::args_of(ctx, pool), src_pages, dst_pages, static_cast<unsigned>(n));
    else lokal::launch_k(lokal::pool_copy_kernel<unsigned short>, grid, 256, 0, st, lokal::args_of(ctx, pool), src_pages, dst_pages, static_cast<unsigned>(n));
    LOKAL_CHECK_LAUNCH(ctx, "pool_copy_kernel");
    return LOKAL_OK;
}

int lokal_cuda_kv_pool_accept(lokal_cuda_ctx* ctx, lokal_cuda_stream s, lokal_kv_pool* pool, const uint32_t* slots,
                              const int32_t* q_start, const int32_t* accepted, const int32_t* n_accepted, uint32_t max_accept,
                              size_t n_seqs) {
    LOKAL_POOL_ENTER(ctx, pool, "kv_pool_accept");
    int rc = lokal::check_list(ctx, pool, "kv_pool_accept", n_seqs, q_start, n_accepted, true);
    if (rc != LOKAL_OK) return rc;
    if (max_accept > lokal::kMaxAccept) return ctx->fail(LOKAL_ERR_BAD_ARG, "kv_pool_accept: max_accept %u is above %u", max_accept, lokal::kMaxAccept);
    if (n_seqs && max_accept && !accepted) return ctx->fail(LOKAL_ERR_BAD_ARG, "kv_pool_accept: a list is null");
    if (!lokal::aligned_to(slots, 4) || !lokal::aligned_to(accepted, 4)) return ctx->fail(LOKAL_ERR_MISALIGNED, "kv_pool_accept: a list is not 4-byte aligned");
    if (n_seqs == 0) return LOKAL_OK;
    cudaStream_t st = static_cast<cudaStream_t>(s);
    const lokal::AcceptArgs t{slots, q_start, accepted, n_accepted, static_cast<unsigned>(n_seqs), max_accept};
    const unsigned long long vecs = pool->a.row_bytes / (pool->vec16 ? 16 : 2) * pool->a.n_stores;
    const dim3 grid(static_cast<unsigned>((vecs + 255) / 256 < 1024 ? (vecs + 255) / 256 : 1024), static_cast<unsigned>(n_seqs));
    if (pool->vec16) lokal::launch_k(lokal::pool_accept_kernel<uint4>, grid, 256, 0, st, lokal::args_of(ctx, pool), t);
    else lokal::launch_k(lokal::pool_accept_kernel<unsigned short>, grid, 256, 0, st, lokal::args_of(ctx, pool), t);
    LOKAL_CHECK_LAUNCH(ctx, "pool_accept_kernel");
    return LOKAL_OK;
}

}  // extern "C"
