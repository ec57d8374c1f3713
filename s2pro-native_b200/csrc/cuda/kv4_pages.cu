/* Paged 4-bit cache: page tables, reference counts and the pages themselves.
 *
 * The decisions (which page goes to whom) are integer scans by one CTA: free pages are taken lowest first and handed out in
 * the order of the call, so the outcome does not depend on timing.  The bytes move in a second kernel over all SMs, bound by HBM
 * (24 pages of 36 layers and 8 kv heads, 71 MB read and written: 22.0 us with the decisions, 6.4 TB/s). */
#include "kv4.cuh"

namespace s2p {

constexpr int KV4_SCAN_THREADS = 1024, KV4_SCAN_WARPS = KV4_SCAN_THREADS / 32;
constexpr int KV4_SCAN_PAGES = 4 * KV4_SCAN_THREADS; /* pages looked at per round */

/* the page operators' part of the workspace: words[0] pages to move; then pairs (from, to); then new numbers */
struct Kv4Lists {
    int* words;
    int2* moves;
    int* renumber;
};
static_assert(256 + ((size_t)KV4_MAX_PAGES / 2 + 1 + S2P_B200_KV4_MAX_LIST) * sizeof(int2) + (size_t)KV4_MAX_PAGES * sizeof(int) <= KV4_AREA_BYTES, "the lists");
static inline Kv4Lists kv4_lists(const s2p_b200_kv4& c) {
    unsigned char* at = static_cast<unsigned char*>(c.work) + KV4_STATUS_BYTES;
    Kv4Lists l;
    l.words = reinterpret_cast<int*>(at);
    l.moves = reinterpret_cast<int2*>(at + 256);
    l.renumber = reinterpret_cast<int*>(l.moves + c.n_pages / 2 + 1 + S2P_B200_KV4_MAX_LIST);
    return l;
}

/* sum over all threads before this one; the total to `total`.  Every thread of the CTA calls it. */
template <class T> __device__ __forceinline__ T kv4_scan(T v, T& total, T* sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    T incl = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const T o = __shfl_up_sync(S2P_FULL_MASK, incl, off);
        if (lane >= off) incl += o;
    }
    if (lane == 31) sh[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        const T w = sh[lane];
        T wi = w;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const T o = __shfl_up_sync(S2P_FULL_MASK, wi, off);
            if (lane >= off) wi += o;
        }
        sh[lane] = wi - w;
        if (lane == 31) sh[32] = wi;
    }
    __syncthreads();
    const T before = sh[warp] + incl - v;
    total = sh[32];
    __syncthreads();
    return before;
}

/* references of pages p .. p + 3; 1 (in use) behind the pool's end */
__device__ __forceinline__ int4 kv4_refs4(const int32_t* refs, int p, int n) {
    if (p + 4 <= n && (reinterpret_cast<uintptr_t>(refs) & 15) == 0) return __ldcg(reinterpret_cast<const int4*>(refs + p));
    return make_int4(p < n ? __ldcg(refs + p) : 1, p + 1 < n ? __ldcg(refs + p + 1) : 1, p + 2 < n ? __ldcg(refs + p + 2) : 1,
                     p + 3 < n ? __ldcg(refs + p + 3) : 1);
}
__device__ __forceinline__ int kv4_count_free(const int32_t* refs, int n, int* sh) {
    int mine = 0, total;
    for (int p = 4 * (int)threadIdx.x; p < n; p += KV4_SCAN_PAGES) {
        const int4 r = kv4_refs4(refs, p, n);
        mine += (r.x == 0) + (r.y == 0) + (r.z == 0) + (r.w == 0);
    }
    kv4_scan(mine, total, sh);
    return total;
}
/* give(rank, page) for the lowest `wanted` free pages, by some thread of the CTA */
template <class Give> __device__ __forceinline__ void kv4_each_free(const int32_t* refs, int n, int wanted, int* sh, Give give) {
    for (int base = 0, seen = 0; base < n && seen < wanted; base += KV4_SCAN_PAGES) {
        const int p = base + 4 * (int)threadIdx.x;
        const int4 r = kv4_refs4(refs, p, n);
        const int f[4] = {r.x == 0, r.y == 0, r.z == 0, r.w == 0};
        int total, rank = seen + kv4_scan(f[0] + f[1] + f[2] + f[3], total, sh);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (f[i]) {
                if (rank < wanted) give(rank, p + i);
                rank++;
            }
        seen += total;
    }
}

struct Kv4Book {
    int32_t *table, *lens, *refs;
    int n_pages, max_seqs, stride;
};
static inline Kv4Book kv4_book(const s2p_b200_kv4& c) { return Kv4Book{c.table, c.lens, c.refs, c.n_pages, c.max_seqs, c.table_stride}; }

__device__ __forceinline__ int kv4_pages_of(int positions) { return positions / S2P_B200_KV4_PAGE + (positions % S2P_B200_KV4_PAGE != 0); }
__device__ __forceinline__ int kv4_held(const Kv4Book& k, int seq) {
    return (int)min((long long)max(__ldcg(k.lens + seq), 0), (long long)k.stride * S2P_B200_KV4_PAGE);
}

__global__ void __launch_bounds__(KV4_SCAN_THREADS) k_kv4_reserve(Kv4Book k, s2p_b200_kv4_batch b, int32_t* info) {
    __shared__ long long wide[33], upto[S2P_B200_KV4_MAX_BATCH]; /* 1024 entries may ask for 2^24 pages each */
    __shared__ int sh[33], first_of[S2P_B200_KV4_MAX_BATCH], seq_of[S2P_B200_KV4_MAX_BATCH];
    constexpr int SLOTS = 2 * S2P_B200_KV4_MAX_BATCH;
    __shared__ int named[SLOTS], first_named[SLOTS]; /* the sequences that stand in the batch, and where first */
    const int e = threadIdx.x;
    for (int i = e; i < SLOTS; i += KV4_SCAN_THREADS) {
        named[i] = -1;
        first_named[i] = S2P_B200_KV4_MAX_BATCH;
    }
    __syncthreads();
    grid_wait();
    grid_release();
    int seq = -1, held = 0, fits = 0, slot = 0;
    long long after = 0, need = 0;
    if (e < b.n) {
        seq = b.seqs[e];
        if ((unsigned)seq < (unsigned)k.max_seqs) {
            slot = (int)((unsigned)seq * 2654435769u >> 16) % SLOTS; /* (2^32 over the golden ratio) */
            for (int there; (there = atomicCAS(&named[slot], -1, seq)) != -1 && there != seq;) slot = (slot + 1) % SLOTS; /* at most half of them are taken */
            atomicMin(&first_named[slot], e);
        }
    }
    __syncthreads();
    if (e < b.n) {
        if ((unsigned)seq < (unsigned)k.max_seqs && first_named[slot] == e) {
            held = kv4_held(k, seq);
            after = (long long)held + max(0, min(b.row0[e + 1], b.rows) - max(b.row0[e], 0));
            fits = after <= (long long)k.stride * S2P_B200_KV4_PAGE;
            need = (after + S2P_B200_KV4_PAGE - 1) / S2P_B200_KV4_PAGE - kv4_pages_of(held);
        }
    }
    long long total;
    const long long before = kv4_scan(need, total, wide);
    const int n_free = total > 0 || info ? kv4_count_free(k.refs, k.n_pages, sh) : 0;
    const int given = fits && (need == 0 || before + need <= n_free);
    if (e < b.n) {
        upto[e] = before + need;
        first_of[e] = kv4_pages_of(held);
        seq_of[e] = given ? seq : -1;
    }
    int n_given;
    kv4_scan(given ? (int)need : 0, n_given, sh); /* (its barriers also publish the arrays) */
    if (n_given > 0) {
        kv4_each_free(k.refs, k.n_pages, (int)min(total, (long long)n_free), sh, [&](int rank, int page) {
            int lo = 0, hi = b.n - 1; /* the first entry with upto > rank: its pages are those ranks */
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (upto[mid] > rank) hi = mid; else lo = mid + 1;
            }
            if (seq_of[lo] < 0) return;
            const int step = rank - (lo ? (int)upto[lo - 1] : 0);
            k.table[(size_t)seq_of[lo] * k.stride + first_of[lo] + step] = page;
            k.refs[page] = 1;
        });
    }
    if (e < b.n) {
        b.pos0[e] = given ? held : -1;
        if (given) k.lens[seq] = (int)after;
    }
    int refused;
    kv4_scan<int>(e < b.n && !given, refused, sh);
    if (info && e == 0) {
        info[0] = n_free - n_given;
        info[1] = refused;
    }
}

extern "C" cudaError_t kv4_reserve(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int32_t* info, cudaStream_t st) {
    return launch_after(k_kv4_reserve, dim3(1), KV4_SCAN_THREADS, 0, st, kv4_book(*c), *b, info);
}

/* empties a sequence, by a group of `width` threads */
__device__ __forceinline__ void kv4_empty(const Kv4Book& k, int seq, int at, int width) {
    int32_t* entries = k.table + (size_t)seq * k.stride;
    const int n = kv4_pages_of(kv4_held(k, seq));
    for (int j = at; j < n; j += width) {
        const int page = entries[j];
        entries[j] = -1;
        if ((unsigned)page < (unsigned)k.n_pages) atomicSub(k.refs + page, 1);
    }
}

struct Kv4SeqList { int32_t seq[S2P_B200_KV4_MAX_LIST]; };
__global__ void __launch_bounds__(128) k_kv4_release(Kv4Book k, Kv4SeqList list) {
    grid_wait();
    grid_release();
    const int seq = list.seq[blockIdx.x];
    kv4_empty(k, seq, threadIdx.x, 128);
    __syncthreads(); /* lens is read by all before it goes */
    if (threadIdx.x == 0) k.lens[seq] = 0;
}

extern "C" cudaError_t kv4_release(const s2p_b200_kv4* c, const int32_t* seqs, int n, cudaStream_t st) {
    Kv4SeqList list;
    for (int i = 0; i < n; i++) list.seq[i] = seqs[i];
    return launch_after(k_kv4_release, dim3((unsigned)n), 128, 0, st, kv4_book(*c), list);
}

struct Kv4ForkList { int32_t parent[S2P_B200_KV4_MAX_LIST], child[S2P_B200_KV4_MAX_LIST], tokens[S2P_B200_KV4_MAX_LIST]; };

/* Tables and references of a fork; the pages to copy go to the lists. */
__global__ void __launch_bounds__(KV4_SCAN_THREADS) k_kv4_fork(Kv4Book k, Kv4ForkList list, int n, Kv4Lists lists, int32_t* info) {
    __shared__ int sh[33], tail_to[S2P_B200_KV4_MAX_LIST], taker[S2P_B200_KV4_MAX_LIST], full_of[S2P_B200_KV4_MAX_LIST];
    grid_wait();
    grid_release();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = threadIdx.x;
    for (int i = warp; i < n; i += KV4_SCAN_WARPS) kv4_empty(k, list.child[i], lane, 32);
    __threadfence();
    __syncthreads();
    int tokens = 0, full = 0, from = -1;
    if (e < n) {
        const int held = kv4_held(k, list.parent[e]);
        tokens = list.tokens[e] < 0 ? held : min(list.tokens[e], held);
        full = tokens / S2P_B200_KV4_PAGE;
        if (tokens % S2P_B200_KV4_PAGE) from = __ldcg(k.table + (size_t)list.parent[e] * k.stride + full);
        if ((unsigned)from >= (unsigned)k.n_pages) from = -1;
        tail_to[e] = -1;
    }
    int n_need, n_given, refused;
    const int rank = kv4_scan<int>(from >= 0, n_need, sh);
    if (from >= 0) taker[rank] = e;
    const int n_free = kv4_count_free(k.refs, k.n_pages, sh);
    if (n_need > 0) /* taker is published by the count's barriers */
        kv4_each_free(k.refs, k.n_pages, min(n_need, n_free), sh, [&](int r, int page) { tail_to[taker[r]] = page; });
    __syncthreads();
    const int given = e < n && (from < 0 || tail_to[e] >= 0);
    if (e < n) {
        full_of[e] = given ? full : 0;
        k.lens[list.child[e]] = given ? tokens : 0;
    }
    const int at = kv4_scan<int>(given && from >= 0, n_given, sh);
    if (given && from >= 0) {
        lists.moves[at] = make_int2(from, tail_to[e]);
        k.table[(size_t)list.child[e] * k.stride + full] = tail_to[e];
        k.refs[tail_to[e]] = 1;
    }
    kv4_scan<int>(e < n && !given, refused, sh);
    for (int i = warp; i < n; i += KV4_SCAN_WARPS) {
        const int32_t* source = k.table + (size_t)list.parent[i] * k.stride;
        int32_t* to = k.table + (size_t)list.child[i] * k.stride;
        for (int j = lane; j < full_of[i]; j += 32) {
            const int page = source[j];
            const bool real = (unsigned)page < (unsigned)k.n_pages;
            to[j] = real ? page : -1;
            if (real) atomicAdd(k.refs + page, 1);
        }
    }
    if (e == 0) {
        lists.words[0] = n_given;
        if (info) {
            info[0] = n_free - n_given;
            info[1] = refused;
        }
    }
}

/* Copies the listed pages, 16 bytes a thread and load, eight loads under way; then, where pages were renumbered, the tables. */
constexpr int KV4_COPY_THREADS = 512, KV4_COPY_UNROLL = 8;
constexpr size_t KV4_COPY_CHUNK = (size_t)KV4_COPY_THREADS * KV4_COPY_UNROLL * 16;
__global__ void __launch_bounds__(KV4_COPY_THREADS) k_kv4_move(unsigned char* pages, size_t page_bytes, Kv4Lists lists, int32_t* table, size_t entries,
                                                               const int* used, int n_pages) {
    grid_wait();
    grid_release();
    const int moves = lists.words[0];
    const size_t per_page = (page_bytes + KV4_COPY_CHUNK - 1) / KV4_COPY_CHUNK;
    for (size_t c = blockIdx.x; c < per_page * (size_t)moves; c += gridDim.x) {
        const int2 mv = lists.moves[c / per_page];
        const size_t off = c % per_page * KV4_COPY_CHUNK + (size_t)threadIdx.x * 16;
        const unsigned char* from = pages + (size_t)mv.x * page_bytes;
        unsigned char* to = pages + (size_t)mv.y * page_bytes;
        uint4 v[KV4_COPY_UNROLL];
#pragma unroll
        for (int i = 0; i < KV4_COPY_UNROLL; i++) {
            const size_t o = off + (size_t)i * KV4_COPY_THREADS * 16;
            if (o < page_bytes) v[i] = __ldcs(reinterpret_cast<const uint4*>(from + o));
        }
#pragma unroll
        for (int i = 0; i < KV4_COPY_UNROLL; i++) {
            const size_t o = off + (size_t)i * KV4_COPY_THREADS * 16;
            if (o < page_bytes) __stcs(reinterpret_cast<uint4*>(to + o), v[i]);
        }
    }
    if (!table || !moves) return;
    const int first = used[0];
    for (size_t i = (size_t)blockIdx.x * KV4_COPY_THREADS + threadIdx.x; i < entries; i += (size_t)gridDim.x * KV4_COPY_THREADS) {
        const int page = table[i];
        if (page >= first && page < n_pages) table[i] = lists.renumber[page];
    }
}
static cudaError_t kv4_move(const s2p_b200_kv4& c, const Kv4Lists& lists, int renumber, size_t most, cudaStream_t st) {
    const size_t page = s2p_b200_kv4_page_bytes(c.layers, c.kv_heads), chunks = (page + KV4_COPY_CHUNK - 1) / KV4_COPY_CHUNK;
    const size_t want = chunks * most;
    const unsigned grid = (unsigned)(want < 592 ? (want ? want : 1) : 592); /* two to four CTAs to each of 148 SMs; the kernel strides */
    return launch_after(k_kv4_move, dim3(grid), KV4_COPY_THREADS, 0, st, static_cast<unsigned char*>(c.pages), page, lists,
                        renumber ? c.table : static_cast<int32_t*>(nullptr), (size_t)c.max_seqs * (size_t)c.table_stride, lists.words + 1, c.n_pages);
}

extern "C" cudaError_t kv4_fork(const s2p_b200_kv4* c, const int32_t* parents, const int32_t* children, const int32_t* tokens, int n, int32_t* info,
                                cudaStream_t st) {
    Kv4ForkList list;
    for (int i = 0; i < n; i++) {
        list.parent[i] = parents[i];
        list.child[i] = children[i];
        list.tokens[i] = tokens[i];
    }
    const Kv4Lists lists = kv4_lists(*c);
    const cudaError_t e = launch_after(k_kv4_fork, dim3(1), KV4_SCAN_THREADS, 0, st, kv4_book(*c), list, n, lists, info);
    return e != cudaSuccess || !n ? e : kv4_move(*c, lists, 0, (size_t)n, st);
}

/* The k-th used page with a number of at least U, the count of used pages, goes to the k-th free one below U; there are as
 * many of the one as of the other. */
__global__ void __launch_bounds__(KV4_SCAN_THREADS) k_kv4_compact(Kv4Book k, Kv4Lists lists, int32_t* info) {
    __shared__ int sh[33];
    grid_wait();
    grid_release();
    const int used = k.n_pages - kv4_count_free(k.refs, k.n_pages, sh);
    int from_seen = 0, to_seen = 0;
    for (int base = 0; base < k.n_pages; base += KV4_SCAN_PAGES) {
        const int p = base + 4 * (int)threadIdx.x;
        const int4 r = kv4_refs4(k.refs, p, k.n_pages);
        const int u[4] = {r.x != 0, r.y != 0, r.z != 0, r.w != 0};
        int from = 0, to = 0, total_from, total_to;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            from += u[i] && p + i >= used && p + i < k.n_pages;
            to += !u[i] && p + i < used;
        }
        int rf = from_seen + kv4_scan(from, total_from, sh), rt = to_seen + kv4_scan(to, total_to, sh);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (u[i] && p + i >= used && p + i < k.n_pages) lists.moves[rf++].x = p + i;
            if (!u[i] && p + i < used) lists.moves[rt++].y = p + i;
            if (p + i >= used && p + i < k.n_pages) lists.renumber[p + i] = p + i; /* a table may name a page that no reference counts */
        }
        from_seen += total_from;
        to_seen += total_to;
    }
    __threadfence_block();
    __syncthreads();
    const int moves = min(from_seen, to_seen);
    for (int i = threadIdx.x; i < moves; i += KV4_SCAN_THREADS) {
        const int2 mv = lists.moves[i];
        lists.renumber[mv.x] = mv.y;
        k.refs[mv.y] = __ldcg(k.refs + mv.x);
        k.refs[mv.x] = 0;
    }
    if (threadIdx.x == 0) {
        lists.words[0] = moves;
        lists.words[1] = used;
        if (info) {
            info[0] = k.n_pages - used;
            info[1] = moves;
        }
    }
}

extern "C" cudaError_t kv4_compact(const s2p_b200_kv4* c, int32_t* info, cudaStream_t st) {
    const Kv4Lists lists = kv4_lists(*c);
    const cudaError_t e = launch_after(k_kv4_compact, dim3(1), KV4_SCAN_THREADS, 0, st, kv4_book(*c), lists, info);
    return e != cudaSuccess ? e : kv4_move(*c, lists, 1, (size_t)c->n_pages / 2, st);
}

}  // namespace s2p
