/* Attention of prompt slices over the paged 4-bit cache, on the 5th-generation tensor cores.
 *
 * A unit is one kv head of one sequence with two tiles of 128 query rows each: 128 / G consecutive rows of the slice times the G
 * query heads of that kv head (32 rows at G = 4).  It walks the sequence page by page:
 *
 *   S = Q K^T    [128 x 64], tcgen05.mma, both operands in shared memory, f32 in TMEM
 *   P = 2^((S - m) f), f16, over columns that held S; running maximum m and sum in 32 bits, m renewed where a score passes it by 8.  (S f - m f, one instruction less a
 *   pair, leaves the rounding of m f as the largest exponent: thousands where queries are large enough.)
 *   O += P V     [128 x 128], P from TMEM, V in shared memory, f32 in TMEM
 *
 * Roles, coupled by mbarriers only:
 *   warps 0..3, 4..7   one thread a query row of the first, second tile: the softmax with the row's 64 scores in registers, at the end the result
 *   warps 8..11, 12..15  every other page each: bring it into shared memory (with loads into registers, one page ahead, they waited for half their
 *                      time; one team of four warps alone took 1.4 us a page, twice what the products need) and turn it into operands: s c + m in f16 (one rounding, 2^-11), keys as [channel / 8][position] units of 8
 *                      channels, values likewise; three stages.  A team also brings a row tile's queries, as f16 (times a power of two, so that
 *                      a row's largest value is 512..1023: exact)
 *   warps 16, 17       one thread each issues a row tile's products.  Each row tile has two places for scores, so the scores of page i + 1 are
 *                      computed while the softmax of page i runs: it never waits for them.
 * Both row tiles use the same converted keys and values, which is what two of them are for.  Every operand is in the unswizzled
 * core-matrix layout (8 rows x 16 bytes); a unit plane has 32 or 16 bytes more than its positions take, so that the converting lanes'
 * stores fall on different banks.
 *
 * The pages of all units, and what each costs besides, form one line, and each CTA takes an equal stretch of it, wherever that cuts units.  With no more units than CTAs
 * most CTAs would get the end of one unit and the start of the next: there every unit is cut into equal parts of its own, one to a CTA
 * (32 query and 8 kv heads, 512 rows behind 1500: 49 -> 41 us when it came, 39.4 now; 77 behind 1024: 30 -> 24.5).  The parts of a
 * unit are added, in order, by a second kernel over all SMs: in the last CTA to arrive that took 8 us for two parts of 128 KB and 20 for
 * five, with the other SMs idle.  Parts stay in 32 bits (f16 would take 1.5 us off the smallest calls).
 * A page takes a CTA 2180 cycles (2048 rows, the last of 8100, 32 query and 8 kv heads: 280 to 306 us at 1.75 to 1.6 GHz, 780 to 850 TFLOP/s); the tensor cores are busy 56% of
 * that, the issue slots 63%: the roles wait for each other's results.  ptxas spills 64 bytes (260 loaded) at 96 registers. */
#include "kv4.cuh"
#include "pipe.cuh"

namespace s2p {

constexpr int KS_ROWS = 128, KS_TILE = S2P_B200_KV4_PAGE, KS_STAGES = 3, KS_RAW = 2, KS_WARPS = 20, KS_THREADS = KS_WARPS * 32, KS_SOFTMAX = 256;
constexpr int KS_Q_PITCH = 128 * 16 + 16, KS_Q_BYTES = 16 * KS_Q_PITCH;                                  /* one row tile: [channel / 8][row] units */
constexpr int KS_K_PITCH = KS_TILE * 16 + 32, KS_V_PITCH = KS_TILE * 16 + 16;
constexpr int KS_K_BYTES = 16 * KS_K_PITCH, KS_V_BYTES = 16 * KS_V_PITCH;
constexpr int KS_OPERANDS = 2 * KS_Q_BYTES + KS_STAGES * (KS_K_BYTES + KS_V_BYTES) + 2 * KS_RAW * KV4_HEAD_BYTES;
constexpr int KS_LEAST = 3;  /* pages that make a CTA worth its while: 77 rows behind 1024 with 2 and 3: 26.9 and 25.2 us; longer calls have more in any case */
/* Pages that a unit costs a CTA besides its own: a prompt's first units have one page, two, ..., and without this a few CTAs get them all.  Prompts of 1000, 2000, 4000 from
 * their first position with 0, 4, 6, 9: 88, 39, 39, 40 us; 190, 88, 83, 83; 431, 236, 200, 202. */
constexpr int KS_UNIT = 6;
constexpr int KS_SECOND = 4; /* pages that a second unit costs a CTA (5 us: queries, a part to write, another's to read) */
static_assert(KS_OPERANDS % 16 == 0 && KS_K_BYTES % 16 == 0 && KS_V_BYTES % 16 == 0, "descriptors count 16 bytes");

struct KsBars {
    uint64_t k_full[KS_STAGES], k_free[KS_STAGES], v_full[KS_STAGES], v_free[KS_STAGES];
    uint64_t s_full[2][2], p_full[2][2]; /* [row tile][place] */
    uint64_t o_done[2], q_full, q_free, unit_done[2], all_done[2];
};

struct KsLine { /* in shared memory: the chunks (units of one kv head each) of all entries */
    unsigned* upto;  /* [chunks + 1] position tiles times kv heads before a chunk */
    int* first;      /* [entries + 1] chunks before an entry */
    int* start;      /* [entries + 1] rows before an entry */
    int *seq, *p0;   /* [entries] its sequence, and its first position or -1 */
};
static inline size_t ks_line_bytes(int chunks, int n) { return (size_t)(chunks + 1 + 4 * (n + 1)) * 4; }

/* What a CTA leaves: slot 2 w + 1 where CTA w begins a unit that others end, 2 w where it goes on with one. */
struct KsParts {
    float *max, *sum; /* [slot][256 rows] */
    float4* o;        /* [slot][column / 4][256 rows] */
    int4* unit;       /* [w] the unit that w begins and others end: first row, rows (0: none), kv head, last CTA */
    int* status;
};
/* Columns of O are the values' channels in the order of their units: unit u holds channels 64 (u / 8) + 4 (u % 8) + 0 .. 3 in its even places and
 * the same + 32 in its odd ones. */

__device__ __forceinline__ uint64_t ks_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) | ((uint64_t)((sbo >> 4) & 0x3FFFu) << 32) | (1ull << 46);
}
__device__ __forceinline__ void ks_ld32(uint32_t addr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(addr) : "memory");
}
__device__ __forceinline__ void ks_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void ks_ld16(uint32_t addr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(addr) : "memory");
}
__device__ __forceinline__ void ks_st16(uint32_t addr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
        ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
          "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(addr) : "memory");
}
__device__ __forceinline__ void ks_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void ks_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void ks_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void ks_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void ks_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
__device__ __forceinline__ void ks_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
/* Waits of this kernel: mbar_wait_bounded (pipe.cuh) with the case that nothing has to be waited for in front and the rest out of its way.  (As it
 * stands there, written out at every place, it cost the issuing thread 0.2 us a wait that was over already: its instructions had to be fetched
 * each time.) */
__device__ __forceinline__ bool ks_wait(uint64_t* bar, unsigned parity, int* status) {
    if (__builtin_expect(mbar_try_wait(bar, parity), 1)) return true;
    const unsigned long long t0 = pipe_now();
    for (unsigned i = 1; !mbar_try_wait(bar, parity); i++)
        if ((i & 7u) == 0 && (status_peek(status) != PIPE_OK || pipe_now() - t0 > c_pipe_wait_ns || i >= PIPE_MBAR_TRIES)) {
            atomicCAS(status, PIPE_OK, PIPE_ERR_TMA_WAIT);
            return false;
        }
    return true;
}
__device__ __forceinline__ bool ks_wait_warp(uint64_t* bar, unsigned parity, int* status) { return __all_sync(S2P_FULL_MASK, ks_wait(bar, parity, status)); }
template <int X> struct KsTile { static constexpr int value = X; };
__device__ __forceinline__ void ks_pages_sync(int team) { asm volatile("bar.sync %0, 128;" ::"r"(1 + team) : "memory"); }
__device__ __forceinline__ float ks_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
/* two at a time; three at a time */
__device__ __forceinline__ float2 ks_mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, r;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 r, x, y;\n\tmov.b64 {%0, %1}, r;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 ks_add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, r;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 r, x, y;\n\tmov.b64 {%0, %1}, r;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float ks_max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ uint32_t ks_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ __half2 ks_h2(uint32_t w) { return *reinterpret_cast<const __half2*>(&w); }
__device__ __forceinline__ uint32_t ks_u(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
/* A group's largest code may stand for more than the 65504 that its largest value was kept at, by the roundings of m (16) and s (fifteen times 4): up to 65580, and from 65520
 * on that is no f16.  m alone does not do it: with s < 32 the code would be 14.  True where one of the four s in x, y (z, w: m) is 32 or more; those operands are kept at
 * 65504 by a second pass over them.  (Operands at half their size need no such pass, but s, m and s c + m below 2^-13 lose their last bit: scores of keys of 1e-5 were 6% off.) */
__device__ __forceinline__ bool ks_wide(const uint4& w) { return (((w.x + 0x30003000u) | (w.y + 0x30003000u)) & 0x80008000u) != 0; }
__device__ __forceinline__ uint32_t ks_keep(uint32_t w) { return ks_u(__hmin2(ks_h2(w), ks_h2(0x7BFF7BFFu))); }
__device__ __forceinline__ void ks_keep(unsigned char* at) {
    uint4* to = reinterpret_cast<uint4*>(at);
    *to = make_uint4(ks_keep(to->x), ks_keep(to->y), ks_keep(to->z), ks_keep(to->w));
}
/* eight codes of a word as s c + m: nibbles 0 and 4, 1 and 5, 2 and 6, 3 and 7 (those of a byte's upper half come as 16 c) */
__device__ __forceinline__ uint4 ks_widen(uint32_t w, __half2 s, __half2 m) {
    const __half2 k1024 = ks_h2(0x64006400u), k16th = ks_h2(0x2C002C00u), k64 = ks_h2(0xD400D400u); /* 1024, 1 / 16, -64 */
    const uint32_t x = w >> 8;
    uint4 r;
    r.x = ks_u(__hfma2(__hsub2(ks_h2((w & 0x000F000Fu) | 0x64006400u), k1024), s, m));
    r.y = ks_u(__hfma2(__hfma2(ks_h2((w & 0x00F000F0u) | 0x64006400u), k16th, k64), s, m));
    r.z = ks_u(__hfma2(__hsub2(ks_h2((x & 0x000F000Fu) | 0x64006400u), k1024), s, m));
    r.w = ks_u(__hfma2(__hfma2(ks_h2((x & 0x00F000F0u) | 0x64006400u), k16th, k64), s, m));
    return r;
}
__device__ __forceinline__ uint32_t ks_word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

/* Entries of up to `few` rows are left to the kernel for single tokens. */
__global__ void __launch_bounds__(KS_THREADS, 1)
k_kv4_slices(Kv4View cache, Kv4Rows b, int few, const __nv_bfloat16* q, __nv_bfloat16* out, KsParts parts) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ KsBars bars;
    __shared__ uint32_t sh_tmem;
    __shared__ float sh_factor[4][KS_SOFTMAX]; /* of the query rows of a unit, four units deep: to base-2 logits */
    __shared__ struct { unsigned begin, end, last, share, more; } sh_line; /* this CTA's stretch; the last CTA of the one unit it has a part of, or 0; all stretches */
    __shared__ int sh_absent[16];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int group = cache.q_heads / cache.kv_heads, tile_rows = KS_ROWS / group, unit_rows = 2 * tile_rows;
    const int capacity = cache.stride * S2P_B200_KV4_PAGE;
    unsigned char *sq = smem, *sk = sq + 2 * KS_Q_BYTES, *sv = sk + KS_STAGES * KS_K_BYTES, *raw = sv + KS_STAGES * KS_V_BYTES;
    KsLine line;
    line.first = reinterpret_cast<int*>(smem + KS_OPERANDS);
    line.start = line.first + b.n + 1;
    line.seq = line.start + b.n + 1;
    line.p0 = line.seq + b.n + 1;
    line.upto = reinterpret_cast<unsigned*>(line.p0 + b.n + 1);
    int* status = parts.status;

    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        for (int i = 0; i < KS_STAGES; i++) {
            mbar_init(&bars.k_full[i], 4);
            mbar_init(&bars.k_free[i], 2);
            mbar_init(&bars.v_full[i], 4);
            mbar_init(&bars.v_free[i], 2);
        }
        for (int i = 0; i < 2; i++) {
            for (int j = 0; j < 2; j++) {
                mbar_init(&bars.s_full[i][j], 1);
                mbar_init(&bars.p_full[i][j], 4);
            }
            mbar_init(&bars.o_done[i], 1);
            mbar_init(&bars.unit_done[i], 1);
            mbar_init(&bars.all_done[i], 1);
        }
        mbar_init(&bars.q_full, 8);
        mbar_init(&bars.q_free, 2);
        mbar_init_fence();
    }
    grid_wait();
    grid_release();
    ks_before_sync();

    auto rows_of = [&](int e) { return line.start[e + 1] - line.start[e]; };
    auto chunks_of = [&](int e) { return rows_of(e) > few ? (rows_of(e) + unit_rows - 1) / unit_rows : 0; };
    auto seen_by = [&](int p0, int row) { return p0 < 0 ? 0 : (int)min((long long)p0 + row + 1, (long long)capacity); };
    auto entry_of = [&](int chunk) { /* the entry whose chunk it is */
        int lo = 0, hi = b.n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (line.first[mid] <= chunk) lo = mid; else hi = mid;
        }
        return lo;
    };
    auto tiles_of = [&](int e, int chunk) { /* pages of a chunk's unit */
        const int last = min(rows_of(e), (chunk - line.first[e] + 1) * unit_rows) - 1;
        return max(1, (seen_by(line.p0[e], last) + KS_TILE - 1) / KS_TILE);
    };
    /* ---- the line of work, by one warp: 32 entries or chunks at a time, so no barrier for the usual few ---- */
    if (warp == 0) {
        int top = 0; /* starts made ascending and kept inside the activations, whatever row0 holds */
        for (int e0 = 0; e0 <= b.n; e0 += 32) {
            const int e = e0 + lane;
            int r = e <= b.n ? min(b.row0[e], b.rows) : 0;
            if (e < b.n) {
                const int seq = b.seqs[e], p0 = b.pos0[e];
                line.seq[e] = seq;
                line.p0[e] = (unsigned)seq < (unsigned)cache.max_seqs && p0 <= (1 << 30) ? p0 : -1;
            }
            r = max(r, top);
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int o = __shfl_up_sync(S2P_FULL_MASK, r, off);
                if (lane >= off) r = max(r, o);
            }
            if (e <= b.n) line.start[e] = r;
            top = __shfl_sync(S2P_FULL_MASK, r, 31);
        }
        __syncwarp();
        auto before = [&](unsigned v, unsigned& carry) { /* carry + the lanes before this one; carry goes on */
            unsigned at = v;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const unsigned o = __shfl_up_sync(S2P_FULL_MASK, at, off);
                if (lane >= off) at += o;
            }
            const unsigned all = __shfl_sync(S2P_FULL_MASK, at, 31), mine = carry + at - v;
            carry += all;
            return mine;
        };
        unsigned chunks = 0, total = 0;
        for (int e0 = 0; e0 <= b.n; e0 += 32) {
            const int e = e0 + lane;
            const unsigned at = before(e < b.n ? (unsigned)chunks_of(e) : 0u, chunks);
            if (e <= b.n) line.first[e] = (int)at;
        }
        __syncwarp();
        int most = 0; /* pages of the longest unit */
        for (int c0 = 0; c0 <= (int)chunks; c0 += 32) {
            const int c = c0 + lane;
            const int t = c < (int)chunks ? tiles_of(entry_of(c), c) : 0;
            most = max(most, t);
            const unsigned at = before(t ? (unsigned)(KS_UNIT + t) * (unsigned)cache.kv_heads : 0u, total);
            if (c <= (int)chunks) line.upto[c] = at;
        }
        most = (int)__reduce_max_sync(S2P_FULL_MASK, (unsigned)most);
        __syncwarp();
        /* As many units as CTAs or fewer: each is cut into parts of at most `longest` pages, the shortest for which there is a CTA to each part; unless a
         * CTA's equal share of the line is shorter by more than a second unit costs it (a part to write, another's to read). */
        const unsigned heads = (unsigned)cache.kv_heads;
        unsigned workers = min(gridDim.x, max(total / (KS_UNIT + KS_LEAST), min(total, 1u))), longest = 0; /* (a stretch longer than what a unit costs has pages) */
        if (chunks * heads <= gridDim.x && chunks) {
            auto parts_at = [&](unsigned l) {
                unsigned n = 0;
                for (int c = lane; c < (int)chunks; c += 32) n += ((line.upto[c + 1] - line.upto[c]) / heads - KS_UNIT + l - 1) / l;
                return __reduce_add_sync(S2P_FULL_MASK, n) * heads;
            };
            unsigned lo = KS_LEAST, hi = max((unsigned)most, (unsigned)KS_LEAST);
            while (lo < hi) {
                const unsigned mid = (lo + hi) / 2;
                if (parts_at(mid) <= gridDim.x) hi = mid;
                else lo = mid + 1;
            }
            if (lo <= total / workers + KS_SECOND) {
                longest = lo;
                workers = 0;
                if (lane == 0) sh_line.begin = sh_line.end = 0;
                __syncwarp();
                for (int c0 = 0; c0 < (int)chunks; c0 += 32) {
                    const int c = c0 + lane;
                    const unsigned t = c < (int)chunks ? (line.upto[c + 1] - line.upto[c]) / heads - KS_UNIT : 0u, cuts = (t + longest - 1) / longest;
                    const unsigned at = before(cuts * heads, workers);
                    if (blockIdx.x >= at && blockIdx.x - at < cuts * heads) {
                        const unsigned head = (blockIdx.x - at) / cuts, cut = blockIdx.x - at - head * cuts, each = t / cuts, over = t - each * cuts;
                        sh_line.begin = line.upto[c] + head * (KS_UNIT + t) + KS_UNIT + each * cut + min(cut, over);
                        sh_line.end = sh_line.begin + each + (cut < over);
                        sh_line.last = blockIdx.x - cut + cuts - 1;
                    }
                }
            }
        }
        if (lane == 0 && !longest) {
            const unsigned share = workers ? total / workers : 1, more = workers ? total - share * workers : 0, w = min(blockIdx.x, workers);
            sh_line.begin = share * w + min(w, more);
            sh_line.end = blockIdx.x < workers ? sh_line.begin + share + (w < more) : sh_line.begin;
            sh_line.last = 0;
            sh_line.share = share;
            sh_line.more = more;
        }
    }
    __syncthreads();
    ks_after_sync();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&sh_tmem);
    const unsigned chunks = (unsigned)line.first[b.n], worker = blockIdx.x;
    const unsigned begin = sh_line.begin;
    unsigned end = sh_line.end;

    struct Segment {
        int e, head, row0, n_rows, seq, p0, seen, t0, t1, tiles, r0; /* pages t0 .. t1 - 1 of `tiles` */
        unsigned next;                                              /* where the stretch's next unit begins */
    };
    int chunk_at = 0;
    if (begin < end) {
        int lo = 0, hi = (int)chunks;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (line.upto[mid] <= begin) lo = mid; else hi = mid;
        }
        chunk_at = lo;
    }
    if (begin < end) { /* a stretch may end before the first page of its last unit */
        int lo = chunk_at, hi = (int)chunks;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (line.upto[mid] < end) lo = mid; else hi = mid;
        }
        const unsigned inside = end - line.upto[lo], unit = (unsigned)(KS_UNIT + tiles_of(entry_of(lo), lo)), at = inside % unit;
        if (at && at <= (unsigned)KS_UNIT) end -= at;
    }
    auto last_of = [&](const Segment& s, unsigned cur) { /* the last CTA of the unit that this one begins */
        if (sh_line.last) return sh_line.last;
        const unsigned x = cur + (unsigned)s.tiles - 1 /* from its first page */, longer = (sh_line.share + 1) * sh_line.more;
        return x < longer ? x / (sh_line.share + 1) : sh_line.more + (x - longer) / sh_line.share;
    };
    auto segment = [&](unsigned cur, int& chunk) {
        Segment s;
        while (line.upto[chunk + 1] <= cur) chunk++;
        s.e = entry_of(chunk);
        s.tiles = tiles_of(s.e, chunk);
        const unsigned inside = cur - line.upto[chunk];
        const unsigned long_ = (unsigned)(KS_UNIT + s.tiles);
        s.head = (int)(inside / long_);
        const unsigned at = inside - (unsigned)s.head * long_;
        s.next = cur + min(long_ - at, end - cur);
        s.t0 = max((int)at - KS_UNIT, 0);
        s.t1 = (int)(at + (s.next - cur)) - KS_UNIT;
        s.r0 = (chunk - line.first[s.e]) * unit_rows;
        s.n_rows = min(unit_rows, rows_of(s.e) - s.r0);
        s.row0 = line.start[s.e] + s.r0;
        s.seq = line.seq[s.e];
        s.p0 = line.p0[s.e];
        s.seen = seen_by(s.p0, s.r0 + s.n_rows - 1);
        return s;
    };

    const int team = (warp >> 2) & 1, p = tid & 127;
    /* The teams of warps 8..11 and 12..15: each walks along the stretch and brings its pages, one of its own ahead of the conversion. */
    unsigned f_cur = begin, f_it = 0;
    int f_chunk = chunk_at, f_i = 0, page_of = -1; /* lane i keeps the (32 n + i)-th page of the segment */
    Segment f;
    f.t0 = f.t1 = 0;
    auto bring = [&]() { /* the team's next page */
        for (;;) {
            if (f_i == f.t1 - f.t0) {
                if (f_cur == end) break;
                f = segment(f_cur, f_chunk);
                f_cur = f.next;
                f_i = 0;
            }
            if ((f_i & 31) == 0) {
                const int pos = (f.t0 + f_i + lane) * S2P_B200_KV4_PAGE;
                page_of = f_i + lane < f.t1 - f.t0 && pos < f.seen ? kv4_page(cache, f.seq, pos) : -1;
            }
            const int page = __shfl_sync(S2P_FULL_MASK, page_of, f_i & 31);
            const unsigned now = f_it++;
            f_i++;
            if ((int)(now & 1) != team) continue;
            if (page >= 0) {
                const unsigned char* src = kv4_block(cache, page, f.head, 0) + p * 16;
                const uint32_t dst = smem_u32(raw) + (team * KS_RAW + now / 2 % KS_RAW) * KV4_HEAD_BYTES + p * 16;
#pragma unroll
                for (int k = 0; k < KV4_HEAD_BYTES / 2048; k++)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + k * 2048), "l"(src + k * 2048) : "memory");
            }
            if (p == 0) sh_absent[now & 15] = page < 0;
            break;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    /* The query rows of a unit from row tile `tile`, a row to half a warp (a lane has 16 bytes of it), eight rows' loads under way; `first` and `step`:
     * what rows are this half warp's. */
    const unsigned by_group = (65536u + (unsigned)group - 1) / (unsigned)group; /* r / group = r by_group >> 16 for r < 128 */
    auto queries = [&](const Segment& s, unsigned unit, int tile, int first, int step) {
        if (s.n_rows <= tile * tile_rows) return;
        const int u = lane & 15;
        for (int r0 = first; r0 < KS_ROWS; r0 += 8 * step) {
            uint4 w[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int r = r0 + k * step, in = (int)((unsigned)r * by_group >> 16), row = tile * tile_rows + in;
                w[k] = make_uint4(0, 0, 0, 0);
                if (in < tile_rows && row < s.n_rows && r < KS_ROWS)
                    w[k] = reinterpret_cast<const uint4*>(q + ((size_t)(s.row0 + row) * cache.q_heads + (s.head * group + r - in * group)) * 128)[u];
            }
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int r = r0 + k * step;
                /* the largest magnitude of the row, by the bits */
                uint32_t big = __vmaxu2(__vmaxu2(w[k].x & 0x7FFF7FFFu, w[k].y & 0x7FFF7FFFu), __vmaxu2(w[k].z & 0x7FFF7FFFu, w[k].w & 0x7FFF7FFFu));
#pragma unroll
                for (int off = 1; off < 16; off <<= 1) big = __vmaxu2(big, __shfl_xor_sync(S2P_FULL_MASK, big, off));
                const int largest = (int)max(big & 0xFFFFu, big >> 16), e = largest ? min(136 - (largest >> 7), 120) : 0; /* 2^9 <= it times 2^e < 2^10 */
                const float up = __uint_as_float((uint32_t)(127 + e) << 23);
                if (r < KS_ROWS) {
                    if (u == 0) /* log2(e) / sqrt(128) 2^-e */
                        sh_factor[unit & 3][tile * KS_ROWS + r] = __uint_as_float((uint32_t)(127 - e) << 23) * (1.4426950408889634f * 0.08838834764831845f);
                    uint4 h; /* channels 0, 4, 1, 5, 2, 6, 3, 7 of the unit of eight, as ks_widen puts them */
                    h.x = ks_half2(bf_lo(w[k].x) * up, bf_lo(w[k].z) * up);
                    h.y = ks_half2(bf_hi(w[k].x) * up, bf_hi(w[k].z) * up);
                    h.z = ks_half2(bf_lo(w[k].y) * up, bf_lo(w[k].w) * up);
                    h.w = ks_half2(bf_hi(w[k].y) * up, bf_hi(w[k].w) * up);
                    *reinterpret_cast<uint4*>(sq + tile * KS_Q_BYTES + u * KS_Q_PITCH + r * 16) = h;
                }
            }
        }
        fence_proxy_async_smem();
    };
    if (begin < end) {
        if (warp >= 8 && warp < 16) /* the first pages are under way while everybody brings the first unit's queries */
            for (int i = 0; i < KS_RAW - 1; i++) bring();
        int chunk = chunk_at;
        const Segment s = segment(begin, chunk);
        if (warp < 16) queries(s, 0, warp >> 3, (warp & 7) * 2 + (lane >> 4), 16);
    }
    __syncthreads();

    if (warp < 8) {
        /* ================= softmax ================= */
        asm volatile("setmaxnreg.inc.sync.aligned.u32 136;");
        const int x = warp >> 2, r = tid & 127; /* row tile, row */
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t t_o = tmem + (uint32_t)(x * 128) + lanes, t_s = tmem + 256u + (uint32_t)(x * 128) + lanes;
        unsigned n_s = 0, segments = 0, units = 0; /* pages of this row tile so far; units; those in which it has rows */
        bool ok = true, begun = false;
        int chunk = chunk_at;
        unsigned it = 0; /* pages of the CTA so far */
        for (unsigned cur = begin; cur < end && ok;) {
            const Segment s = segment(cur, chunk);
            const int my_row = x * tile_rows + r / group, my_head = s.head * group + r % group;
            const bool live = r < tile_rows * group && my_row < s.n_rows, active = x * tile_rows < s.n_rows;
            const size_t at = ((size_t)(s.row0 + my_row) * cache.q_heads + my_head) * 128;
            float f = 0.0f; /* (there with the first scores, which were issued behind it) */
            const int limit = live ? seen_by(s.p0, s.r0 + my_row) : s.seen;
            float top = -INFINITY, sum = 0.0f;
            if (active)
                for (int i = s.t0; i < s.t1; i++, n_s++) {
                    const unsigned place = n_s & 1;
                    ok = ks_wait_warp(&bars.s_full[x][place], (n_s >> 1) & 1, status);
                    if (!ok) break;
                    ks_after_sync();
                    if (i == s.t0) f = *reinterpret_cast<volatile float*>(&sh_factor[segments & 3][tid]);
                    uint32_t v[2][32];
                    ks_ld32(t_s + 64 * place, v[0]);
                    ks_ld32(t_s + 64 * place + 32, v[1]);
                    const int left = *reinterpret_cast<volatile int*>(&sh_absent[(it + (unsigned)(i - s.t0)) & 15]) ? 0 : limit - i * KS_TILE;
                    ks_ld_wait();
                    if (__any_sync(S2P_FULL_MASK, left < KS_TILE)) {
#pragma unroll
                        for (int k = 0; k < 64; k++)
                            if (k >= left) v[k >> 5][k & 31] = 0xFF800000u;
                    }
                    float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int k = 0; k < 64; k += 2) m4[(k >> 1) & 3] = ks_max3(m4[(k >> 1) & 3], __uint_as_float(v[k >> 5][k & 31]), __uint_as_float(v[k >> 5][(k + 1) & 31]));
                    const float most = ks_max3(ks_max3(m4[0], m4[1], m4[2]), m4[3], m4[3]);
                    if (__any_sync(S2P_FULL_MASK, (most - top) * f > 8.0f)) {
                        const float now = fmaxf(most, top), shrink = now == -INFINITY ? 1.0f : ks_exp2((top - now) * f);
                        top = now;
                        sum *= shrink;
                        if (i > s.t0) { /* behind the product of the page before; the one before that was waited for in front of these scores */
                            ok = ks_wait_warp(&bars.o_done[x], (n_s - 1) & 1, status);
                            if (!ok) break;
                            ks_after_sync();
#pragma unroll 1
                            for (int c = 0; c < 8; c++) {
                                uint32_t o[16];
                                ks_ld16(t_o + 16 * c, o);
                                ks_ld_wait();
#pragma unroll
                                for (int k = 0; k < 16; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * shrink);
                                ks_st16(t_o + 16 * c, o);
                            }
                        }
                    }
                    const float base = top == -INFINITY ? 0.0f : top;
                    const float2 f2 = make_float2(f, f), minus = make_float2(-base, -base);
                    float2 s2[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        uint32_t p[16];
#pragma unroll
                        for (int k = 0; k < 16; k++) {
                            const float2 a = ks_mul2(ks_add2(make_float2(__uint_as_float(v[h][2 * k]), __uint_as_float(v[h][2 * k + 1])), minus), f2);
                            const float2 w = make_float2(ks_exp2(a.x), ks_exp2(a.y));
                            s2[k & 1] = ks_add2(s2[k & 1], w);
                            p[k] = ks_half2(w.x, w.y);
                        }
                        ks_st16(t_s + 64 * place + 16 * h, p); /* over scores that are in registers */
                    }
                    if (!ok) break;
                    const float2 both = ks_add2(s2[0], s2[1]);
                    sum += both.x + both.y;
                    /* A query with an infinity makes scores infinite by the keys' signs, or NaN.  Where all that a row sees are -infinity it would look like one that sees
                     * nothing, and that is zeros: */
                    if (left > 0 && top == -INFINITY) sum = __uint_as_float(0x7FFFFFFFu);
                    ks_st_wait();
                    ks_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars.p_full[x][place]);
                }
            it += (unsigned)(s.t1 - s.t0);
            /* The unit's last product of this row tile.  A barrier for each tile, of the units in which it has rows: an issuer without any is done with its unit, and
             * with the next, before the other one is.  (Its next phase needs this tile's weights, so it is never two ahead.) */
            if (ok && active) {
                ok = ks_wait_warp(&bars.unit_done[x], units++ & 1, status);
                ks_after_sync();
            }
            segments++;
            if (!ok) break; /* the other warps' waits give up by themselves: the status word is set */

            const bool whole = s.t0 == 0 && s.t1 == s.tiles;
            auto store = [&](int c, const float (&v)[32]) { /* columns 32 c ..: units 4 c .. 4 c + 3 of values, two groups in turn */
                __nv_bfloat16* to = out + at + 64 * (c >> 1) + 16 * (c & 1);
#pragma unroll
                for (int odd = 0; odd < 2; odd++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        uint32_t w[4];
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const int at0 = 16 * h + 4 * k + odd; /* unit 2 h + k / 2, channels 2 (k % 2), + 1 */
                            const __nv_bfloat162 y = __floats2bfloat162_rn(v[at0], v[at0 + 2]);
                            w[k] = *reinterpret_cast<const uint32_t*>(&y);
                        }
                        *reinterpret_cast<uint4*>(to + 32 * odd + 8 * h) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
            };
            const size_t slot = 2 * (size_t)worker + (s.t0 == 0 ? 1 : 0);
            if (active) {
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    uint32_t v[32];
                    ks_ld32(t_o + 32 * c, v);
                    ks_ld_wait();
                    float y[32];
                    const float scale = !whole ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
                    for (int k = 0; k < 32; k++) y[k] = __uint_as_float(v[k]) * scale;
                    if (whole) {
                        if (live) store(c, y);
                    } else if (live) {
#pragma unroll
                        for (int k = 0; k < 8; k++) parts.o[(slot * 32 + 8 * c + k) * KS_SOFTMAX + tid] = make_float4(y[4 * k], y[4 * k + 1], y[4 * k + 2], y[4 * k + 3]);
                    }
                }
                ks_before_sync(); /* the next unit's first product writes where this has been read */
                if (!whole && live) {
                    parts.max[slot * KS_SOFTMAX + tid] = top == -INFINITY ? top : top * f; /* (without a page f is not there) */
                    parts.sum[slot * KS_SOFTMAX + tid] = sum;
                }
            }
            if (tid == 0 && s.t0 == 0 && !whole) parts.unit[worker] = make_int4(s.row0, s.n_rows, s.head, (int)last_of(s, s.next - (unsigned)s.t1));
            begun |= s.t0 == 0 && !whole;
            cur = s.next;
        }
        if (tid == 0 && !begun) parts.unit[blockIdx.x] = make_int4(0, 0, 0, 0);
    } else if (warp >= 8 && warp < 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        /* ================= pages to operands ================= */
        const int g = lane >> 2, t = lane & 3, plane = (p >> 5) & 1;
        bool ok = true;
        unsigned it = 0, segments = 0;
        int chunk = chunk_at;
        for (unsigned cur = begin; cur < end; segments++) { /* (to its end whatever gave up: a team's warps meet at every page) */
            const Segment s = segment(cur, chunk);
            /* The queries of a unit go where the unit's before were as soon as its last scores are complete, while its last softmax and its result
             * are still to come; behind the team's first page of the unit, which waits for less. */
            bool have_q = segments == 0;
            auto next_queries = [&]() {
                ok = ok && ks_wait_warp(&bars.q_free, (segments - 1) & 1, status);
                if (ok) {
                    queries(s, segments, team, (warp & 3) * 2 + (lane >> 4), 8);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars.q_full);
                }
                have_q = true;
            };
            for (int i = s.t0; i < s.t1; i++, it++) {
                if ((int)(it & 1) != team) continue;
                const unsigned stage = it % KS_STAGES, turn = it / KS_STAGES; /* the turn-th use of the stage */
                asm volatile("cp.async.wait_group %0;" ::"n"(KS_RAW - 2) : "memory");
                ks_pages_sync(team); /* everybody's share of this page has come, and everybody is done with the one before it: */
                bring();         /* ... its place is free */
                const bool absent = *reinterpret_cast<volatile int*>(&sh_absent[it & 15]) != 0;
                const unsigned char* page = raw + (team * KS_RAW + it / 2 % KS_RAW) * KV4_HEAD_BYTES;
                /* a wait that has given up once is not waited for again, but the barriers above need every warp */
                ok = ok && (turn == 0 || ks_wait_warp(&bars.k_free[stage], (turn - 1) & 1, status));
                unsigned char* to = sk + stage * KS_K_BYTES;
                if (ok) {
                    bool wide = false;
#pragma unroll 1
                    for (int j = 0; j < 2; j++) { /* this thread's units are in blocks p >> 6 and 2 + (p >> 6) */
                        const unsigned char* blk = page + (2 * j + (p >> 6)) * KV4_BLOCK_BYTES;
                        const uint4 kc = *reinterpret_cast<const uint4*>(blk + plane * 512 + lane * 16), kp = *reinterpret_cast<const uint4*>(blk + KV4_PARAMS_K + (plane * 8 + g) * 16);
                        const int pos = (2 * j + (p >> 6)) * 16 + plane * 8 + g;
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const uint32_t sw = k < 2 ? kp.x : kp.y, mw = k < 2 ? kp.z : kp.w;
                            const __half2 sc = ks_h2(prmt(sw, sw, (k & 1) ? 0x3232 : 0x1010)), mn = ks_h2(prmt(mw, mw, (k & 1) ? 0x3232 : 0x1010));
                            *reinterpret_cast<uint4*>(to + (4 * k + t) * KS_K_PITCH + pos * 16) = ks_widen(ks_word(kc, k), sc, mn);
                        }
                        wide |= ks_wide(kp);
                    }
                    if (__builtin_expect(wide, 0))
#pragma unroll 1
                        for (int k = 0; k < 8; k++) ks_keep(to + (4 * (k & 3) + t) * KS_K_PITCH + ((k >> 2) * 32 + (p >> 6) * 16 + plane * 8 + g) * 16);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars.k_full[stage]);
                }
                ok = ok && (turn == 0 || ks_wait_warp(&bars.v_free[stage], (turn - 1) & 1, status));
                to = sv + stage * KS_V_BYTES;
                if (ok) {
                    bool wide = false;
#pragma unroll 1
                    for (int j = 0; j < 2; j++) {
                        const unsigned char* blk = page + (2 * j + (p >> 6)) * KV4_BLOCK_BYTES;
                        const uint4 vc = *reinterpret_cast<const uint4*>(blk + 1024 + plane * 512 + lane * 16);
                        const uint4 vs = *reinterpret_cast<const uint4*>(blk + KV4_PARAMS_V + (plane * 4 + t) * 16),
                                    vm = *reinterpret_cast<const uint4*>(blk + KV4_PARAMS_V + 128 + (plane * 4 + t) * 16);
                        const int pos = (2 * j + (p >> 6)) * 16 + plane * 8 + 2 * t;
#pragma unroll
                        for (int k = 0; k < 4; k++) { /* positions pos, pos + 1; words of groups 0, 1 and 2, 3 */
                            const int word = k & 1, second = k >> 1;
                            const uint32_t sel = second ? 0x7632 : 0x5410;
                            const __half2 sc = ks_h2(prmt(word ? vs.z : vs.x, word ? vs.w : vs.y, sel));
                            const __half2 mn = ks_h2(prmt(word ? vm.z : vm.x, word ? vm.w : vm.y, sel));
                            uint4 v = ks_widen(ks_word(vc, 2 * second + word), sc, mn);
                            /* nobody has written what lies behind the last position: it must not meet a zero weight as NaN */
                            if (absent || i * KS_TILE + pos + second >= s.seen) v = make_uint4(0, 0, 0, 0);
                            *reinterpret_cast<uint4*>(to + (g + 8 * word) * KS_V_PITCH + (pos + second) * 16) = v;
                        }
                        wide |= ks_wide(vs) | ks_wide(make_uint4(vs.z, vs.w, 0, 0));
                    }
                    if (__builtin_expect(wide, 0))
#pragma unroll 1
                        for (int k = 0; k < 8; k++) ks_keep(to + (g + 8 * (k & 1)) * KS_V_PITCH + ((k >> 2) * 32 + (p >> 6) * 16 + plane * 8 + 2 * t + (k >> 1 & 1)) * 16);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars.v_full[stage]);
                }
                if (!have_q) next_queries();
            }
            if (!have_q) next_queries();
            cur = s.next;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp >= 16) {
        /* ================= the products ================= */
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        /* D f32, A and B f16, M 128, N 64 and 128; B of the second product has its rows (positions) along K: MN-major */
        const uint32_t idesc = (1u << 4) | (8u << 17) | (8u << 24), idesc_v = (1u << 4) | (16u << 17) | (8u << 24) | (1u << 16);
        /* A warp for each row tile, with a copy of the code each: with the tile as a variable the compiler keeps what the products take in ordinary
         * registers and needs twice their time to issue them; and one warp for both waits for the one tile's weights while the other's are
         * ready (1.4 us a page, the products 0.7). */
        auto issue = [&](auto tile) {
            constexpr int x = decltype(tile)::value;
            const uint64_t dq = ks_desc(smem_u32(sq) + x * KS_Q_BYTES, KS_Q_PITCH, 128), dk = ks_desc(smem_u32(sk), KS_K_PITCH, 128);
            const uint64_t dv = ks_desc(smem_u32(sv), 128, KS_V_PITCH);
            unsigned stage = 0, turn = 0, n = 0, segments = 0; /* n: pages whose values have been asked for */
            bool ok = true;
            int chunk = chunk_at;
            auto place = [&](unsigned page) { return tmem + 256u + x * 128 + 64u * (page & 1); };
            auto scores = [&](unsigned page, unsigned from) {
                const uint32_t d = place(page);
                const uint64_t keys = dk + (uint64_t)(from * (KS_K_BYTES >> 4));
#pragma unroll
                for (int k = 0; k < 8; k++) ks_mma_ss(d, dq + (uint64_t)((k * 2 * KS_Q_PITCH) >> 4), keys + (uint64_t)((k * 2 * KS_K_PITCH) >> 4), idesc, k > 0);
                ks_commit(&bars.s_full[x][page & 1]);
                ks_commit(&bars.k_free[from]);
            };
            for (unsigned cur = begin; cur < end && ok; segments++) {
                const Segment s = segment(cur, chunk);
                const int tiles = s.t1 - s.t0;
                const bool active = s.n_rows > x * tile_rows;
                ok = (segments == 0 || ks_wait(&bars.q_full, (segments - 1) & 1, status)) && ks_wait(&bars.k_full[stage], turn & 1, status);
                if (!ok) break;
                ks_after_sync();
                if (active) scores(n, stage);
                else mbar_arrive(&bars.k_free[stage]);
                if (tiles == 1) ks_commit(&bars.q_free);
                for (int i = 0; i < tiles; i++) {
                    const unsigned next = stage + 1 == KS_STAGES ? 0 : stage + 1, next_turn = turn + (stage + 1 == KS_STAGES);
                    /* The next scores, of this unit or of the one behind it, take the place of the weights before these: that product has to be
                     * complete.  (Waited for at every page, or this would fall two phases behind.) */
                    if (active && n >= 1) ok = ks_wait(&bars.o_done[x], (n - 1) & 1, status);
                    if (!ok) break;
                    if (i + 1 < tiles) {
                        ok = ks_wait(&bars.k_full[next], next_turn & 1, status);
                        if (!ok) break;
                        ks_after_sync();
                        if (active) scores(n + 1, next);
                        else mbar_arrive(&bars.k_free[next]);
                        if (i + 2 == tiles) ks_commit(&bars.q_free); /* (arrives at once where nothing is under way) */
                    }
                    ok = ks_wait(&bars.v_full[stage], turn & 1, status);
                    if (ok && active) ok = ks_wait(&bars.p_full[x][n & 1], (n >> 1) & 1, status);
                    if (!ok) break;
                    ks_after_sync();
                    if (active) {
                        const uint32_t d = place(n);
                        const uint64_t from = dv + (uint64_t)(stage * (KS_V_BYTES >> 4));
#pragma unroll
                        for (int k = 0; k < 4; k++) ks_mma_ts(tmem + x * 128, d + 8 * k, from + (uint64_t)((k * 256) >> 4), idesc_v, i > 0 || k > 0);
                        ks_commit(&bars.o_done[x]);
                        ks_commit(&bars.v_free[stage]);
                        n++;
                    } else mbar_arrive(&bars.v_free[stage]);
                    stage = next;
                    turn = next_turn;
                }
                if (ok && active) ks_commit(&bars.unit_done[x]);
                cur = s.next;
            }
            /* TMEM must not be freed under products in flight: they complete by themselves, and this waits for them with a limit of its own */
            ks_commit(&bars.all_done[x]);
            PipeDeadline dl;
            for (unsigned i = 0; i < PIPE_MBAR_TRIES && !mbar_try_wait(&bars.all_done[x], 0); i++)
                if ((i & 63u) == 63u && dl.expired(2000000000ull)) break;
        };
        if (begin < end && warp < 18 && warp_elect()) {
            if (warp == 16) issue(KsTile<0>());
            else issue(KsTile<1>());
        }
        __syncwarp();
    }
    ks_before_sync();
    __syncthreads();
    ks_after_sync();
    if (warp == 16) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

/* The parts of shared units, in order of the CTAs that left them.  Block (w, y): 32 rows of the unit that CTA w began; a thread has one unit of eight
 * columns of a row, and four parts' loads are under way at a time (eight: the same). */
constexpr int KS_JOIN_ROWS = 32, KS_JOIN_THREADS = 16 * KS_JOIN_ROWS, KS_JOIN_PARTS = 4;
__global__ void __launch_bounds__(KS_JOIN_THREADS) k_kv4_join(KsParts parts, int q_heads, int group, __nv_bfloat16* out) {
    grid_wait();
    grid_release();
    const int w0 = blockIdx.x, r = blockIdx.y * KS_JOIN_ROWS + (threadIdx.x % KS_JOIN_ROWS), u = threadIdx.x / KS_JOIN_ROWS;
    const int4 unit = parts.unit[w0];
    const int tile_rows = KS_ROWS / group, x = r / KS_ROWS, in = r % KS_ROWS, row = x * tile_rows + in / group;
    if (in >= tile_rows * group || row >= unit.y) return;
    const int w1 = unit.w;
    float top = -INFINITY, sum = 0.0f, y[8];
#pragma unroll
    for (int k = 0; k < 8; k++) y[k] = 0.0f;
    for (int w = w0; w <= w1; w += KS_JOIN_PARTS) {
        float m[KS_JOIN_PARTS], l[KS_JOIN_PARTS];
        float4 v[KS_JOIN_PARTS][2];
#pragma unroll
        for (int i = 0; i < KS_JOIN_PARTS; i++) {
            m[i] = -INFINITY;
            l[i] = 0.0f;
            v[i][0] = v[i][1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (w + i <= w1) {
                const size_t slot = (size_t)(2 * (w + i) + (w + i == w0));
                m[i] = __ldcg(parts.max + slot * KS_SOFTMAX + r);
                l[i] = __ldcg(parts.sum + slot * KS_SOFTMAX + r);
                v[i][0] = __ldcg(parts.o + (slot * 32 + 2 * u) * KS_SOFTMAX + r);
                v[i][1] = __ldcg(parts.o + (slot * 32 + 2 * u + 1) * KS_SOFTMAX + r);
            }
        }
        float now = top;
#pragma unroll
        for (int i = 0; i < KS_JOIN_PARTS; i++) now = fmaxf(now, m[i]);
        const float base = now == -INFINITY ? 0.0f : now, keep = ks_exp2(top - base);
        sum *= keep;
#pragma unroll
        for (int k = 0; k < 8; k++) y[k] *= keep;
#pragma unroll
        for (int i = 0; i < KS_JOIN_PARTS; i++) {
            const float weight = ks_exp2(m[i] - base);
            sum = fmaf(l[i], weight, sum);
#pragma unroll
            for (int k = 0; k < 2; k++) {
                y[4 * k] = fmaf(v[i][k].x, weight, y[4 * k]);
                y[4 * k + 1] = fmaf(v[i][k].y, weight, y[4 * k + 1]);
                y[4 * k + 2] = fmaf(v[i][k].z, weight, y[4 * k + 2]);
                y[4 * k + 3] = fmaf(v[i][k].w, weight, y[4 * k + 3]);
            }
        }
        top = now;
    }
    const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
    __nv_bfloat16* to = out + ((size_t)(unit.x + row) * q_heads + unit.z * group + in % group) * 128 + 64 * (u >> 3) + 4 * (u & 7);
#pragma unroll
    for (int odd = 0; odd < 2; odd++) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(y[odd] * scale, y[2 + odd] * scale), d = __floats2bfloat162_rn(y[4 + odd] * scale, y[6 + odd] * scale);
        *reinterpret_cast<uint2*>(to + 32 * odd) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&d));
    }
}

/* chunks that the batch can have: its rows in units, and a broken one for each entry */
static int ks_chunks(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b) {
    const int unit = 2 * (KS_ROWS / (c->q_heads / c->kv_heads));
    const long long most = (long long)b->rows / unit + (b->n < b->rows ? b->n : b->rows);
    return most < (1 << 20) ? (int)most : 1 << 20;
}
constexpr int KS_MOST_SMEM = 221 * 1024; /* 227 KB less what is declared in the kernel */

extern "C" cudaError_t kv4_slices_set_wait_ns(unsigned long long ns) { return cudaMemcpyToSymbol(c_pipe_wait_ns, &ns, sizeof(ns)); }

extern "C" int kv4_slices_serve(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b) {
    return KS_OPERANDS + ks_line_bytes(ks_chunks(c, b), b->n) <= (size_t)KS_MOST_SMEM;
}

extern "C" cudaError_t kv4_slices(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int layer, int few, const void* q, void* out, cudaStream_t st) {
    static bool attr_set[64] = {false};
    static int sms[64] = {0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!attr_set[dev]) {
        e = cudaFuncSetAttribute(k_kv4_slices, cudaFuncAttributeMaxDynamicSharedMemorySize, KS_MOST_SMEM);
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev);
        if (e != cudaSuccess) return e;
        attr_set[dev] = true;
    }
    KsParts p;
    unsigned char* area = static_cast<unsigned char*>(c->work) + KV4_STATUS_BYTES;
    p.status = static_cast<int*>(c->work);
    p.o = reinterpret_cast<float4*>(area);
    p.max = reinterpret_cast<float*>(area + (size_t)2 * KV4_SLICE_CTAS * KS_SOFTMAX * 128 * sizeof(float));
    p.sum = p.max + (size_t)2 * KV4_SLICE_CTAS * KS_SOFTMAX;
    p.unit = reinterpret_cast<int4*>(p.sum + (size_t)2 * KV4_SLICE_CTAS * KS_SOFTMAX);
    const int grid = sms[dev] < KV4_SLICE_CTAS ? sms[dev] : KV4_SLICE_CTAS;
    const __nv_bfloat16* qb = static_cast<const __nv_bfloat16*>(q);
    __nv_bfloat16* ob = static_cast<__nv_bfloat16*>(out);
    e = launch_after(k_kv4_slices, dim3((unsigned)grid), KS_THREADS, KS_OPERANDS + ks_line_bytes(ks_chunks(c, b), b->n), st, kv4_view(*c, layer),
                     kv4_rows(*b), few, qb, ob, p);
    if (e != cudaSuccess) return e;
    return launch_after(k_kv4_join, dim3((unsigned)grid, KS_SOFTMAX / KS_JOIN_ROWS), KS_JOIN_THREADS, 0, st, p, c->q_heads, c->q_heads / c->kv_heads, ob);
}

}  // namespace s2p
