/* Attention over the paged 4-bit cache.
 *
 * A unit of work is one kv head of one sequence with up to 8 NT columns: the query heads of that kv head, for as many
 * consecutive rows as fit.  With a code c standing for s c + m in groups of 32 channels,
 *     q . k  =  sum over groups j of  s_j (q . c)_j + m_j (sum of q)_j,
 *     sum_t p_t v_t  =  sum_t (p_t s_tj) c_t + sum_t p_t m_tj,
 * so the codes go into the matrix instructions as they are and nothing is dequantised: a nibble masked out of a 32-bit word IS an
 * f16 number, the subnormal c 2^-24 (or 16 c 2^-24, for the upper one of a byte, and the sixteenth is taken elsewhere: out of the query
 * for keys, out of the result for values).  Per eight codes that is four masks and a shift.
 *
 *   scores   S^T [16 positions x columns]: A = keys of a block of 16 positions as they lie (a lane's 16 bytes hold its
 *            channels of all four groups), B = the query, in f16 after a power of two per column that makes its largest
 *            value 512..1023 (exact: bf16 has 8 bits).  One accumulator per group, scaled by s in 32 bits; the m term is one more
 *            product, m times the sums of q split into two f16.
 *   softmax  running maximum and sum in 32 bits, base 2; the maximum is renewed only when a score passes it by 2, so that a
 *            block normally costs one vote.  p (at most 4) is rounded to f16, 11 bits, for the products.
 *   values   O^T [128 channels x columns]: A = values, the pairs of positions put together by byte permutation, B = p^T, which is
 *            S^T transposed in registers (movmatrix), times s of the group (rounded to f16 once more; at most 4 * 8734).
 *
 * The cache is read once, so what bounds single tokens is HBM.  Work is cut evenly: the blocks of all units form one line, each
 * CTA takes an equal stretch of it, its warps the stretch's blocks in turn through a ring of asynchronous copies of their own; a
 * unit that several CTAs share is put together by the last of them to arrive, in the CTAs' order, so that the result does not
 * depend on timing. */
#include "kv4.cuh"
#include "pipe.cuh"

namespace s2p {

constexpr int KA_WARPS = 8, KA_THREADS = KA_WARPS * 32, KA_RING = 4;
constexpr int KA_RING_BYTES = KA_WARPS * KA_RING * KV4_BLOCK_BYTES;
constexpr int KA_PASS = 4;                                         /* columns merged at a time */
constexpr int KA_MERGE_BYTES = KA_WARPS * KA_PASS * 128 * 4;
constexpr int KA_LEAST = KA_WARPS;                                 /* blocks that make a CTA worth its while */

struct KaBatch { /* in shared memory, [n (+ 1)] */
    long long* upto; /* blocks of all units before entry b */
    int* start;      /* its first row */
};
static inline size_t ka_batch_bytes(int n) { return ((size_t)(n + 1) * 12 + 15) / 16 * 16; }

__device__ __forceinline__ void ka_mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ka_mma8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5}, {%6}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(b0));
}
__device__ __forceinline__ uint32_t ka_transpose(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t ka_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t ka_mul2(uint32_t a, uint32_t b) {
    const __half2 h = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float ka_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float2 ka_halves(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ uint32_t ka_word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

/* The query of a warp's unit in the layout of the B operands, and what its columns are scaled by. */
template <int NT> struct KaQuery {
    uint32_t b[NT][4][2][2]; /* [column tile][group][half of the group][register] */
    uint32_t sum[NT];        /* sums of q per group, high and low part */
    float factor[NT][2];     /* of the lane's two score columns: to base-2 logits */
};
template <int NT>
__device__ __forceinline__ void ka_load_query(KaQuery<NT>& z, const __nv_bfloat16* q, size_t row_stride, int group, int columns, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int col = nt * 8 + g;
        uint4 raw[4];
#pragma unroll
        for (int j = 0; j < 4; j++) raw[j] = make_uint4(0, 0, 0, 0);
        if (col < columns) {
            const uint4* p = reinterpret_cast<const uint4*>(q + (size_t)(col / group) * row_stride + (size_t)(col % group) * 128) + t;
#pragma unroll
            for (int j = 0; j < 4; j++) raw[j] = p[4 * j]; /* channels 32 j + 8 t .. + 7 */
        }
        float big = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) big = fmaxf(big, fmaxf(fabsf(bf_lo(ka_word(raw[j], i))), fabsf(bf_hi(ka_word(raw[j], i)))));
        big = fmaxf(big, __shfl_xor_sync(S2P_FULL_MASK, big, 1));
        big = fmaxf(big, __shfl_xor_sync(S2P_FULL_MASK, big, 2));
        /* exponent e with 2^9 <= big 2^e < 2^10; 0 for a column of zeros.  e = 136 - E stays in the range of a float's exponents for E >= 10 */
        const int E = (int)(__float_as_uint(big) >> 23);
        const int e = big > 0.0f ? min(136 - E, 120) : 0;
        const float up = __uint_as_float((uint32_t)(127 + e) << 23), down = __uint_as_float((uint32_t)(127 - e) << 23);
        float sums[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float x[8];
            sums[j] = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x[2 * i] = bf_lo(ka_word(raw[j], i)) * up;
                x[2 * i + 1] = bf_hi(ka_word(raw[j], i)) * up;
            }
#pragma unroll
            for (int i = 0; i < 8; i++) sums[j] += x[i];
            z.b[nt][j][0][0] = ka_half2(x[0], x[4]);
            z.b[nt][j][0][1] = ka_half2(x[1] * 0.0625f, x[5] * 0.0625f);
            z.b[nt][j][1][0] = ka_half2(x[2], x[6]);
            z.b[nt][j][1][1] = ka_half2(x[3] * 0.0625f, x[7] * 0.0625f);
            sums[j] += __shfl_xor_sync(S2P_FULL_MASK, sums[j], 1);
            sums[j] += __shfl_xor_sync(S2P_FULL_MASK, sums[j], 2);
        }
        float lo = (t & 1) ? sums[2] : sums[0], hi = (t & 1) ? sums[3] : sums[1];
        if (t & 2) {
            lo -= __half2float(__float2half_rn(lo));
            hi -= __half2float(__float2half_rn(hi));
        }
        z.sum[nt] = ka_half2(lo, hi);
        const float f = down * (1.4426950408889634f * 0.08838834764831845f); /* log2(e) / sqrt(128) */
        z.factor[nt][0] = __shfl_sync(S2P_FULL_MASK, f, 8 * t);
        z.factor[nt][1] = __shfl_sync(S2P_FULL_MASK, f, 8 * t + 4);
    }
}

template <int NT> struct KaState {
    float o[NT][8][4]; /* [column tile][channel tile 2 j + h]: rows 4 g + 2 h (16 times 2^-24 that of the second) and + 1 of group j */
    float om[NT][4];   /* rows g < 4: sum of p m of group g */
    float max[NT][2], sum[NT][2];
};
template <int NT> __device__ __forceinline__ void ka_clear(KaState<NT>& z) {
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) z.o[nt][i][r] = 0.0f;
#pragma unroll
        for (int r = 0; r < 4; r++) z.om[nt][r] = 0.0f;
        z.max[nt][0] = z.max[nt][1] = -INFINITY;
        z.sum[nt][0] = z.sum[nt][1] = 0.0f;
    }
}

/* One block of 16 positions from shared memory.  `left[..]`: positions of the block that each of the lane's columns sees. */
template <int NT, bool MASKED>
__device__ __forceinline__ void ka_block(KaState<NT>& z, const KaQuery<NT>& q, const unsigned char* blk, const int (&left)[NT][2], int lane) {
    const int g = lane >> 2, t = lane & 3;
    const uint4 k0 = *reinterpret_cast<const uint4*>(blk + lane * 16), k1 = *reinterpret_cast<const uint4*>(blk + 512 + lane * 16);
    const uint2 sk0 = *reinterpret_cast<const uint2*>(blk + KV4_PARAMS_K + g * 16), sk1 = *reinterpret_cast<const uint2*>(blk + KV4_PARAMS_K + 128 + g * 16);
    const uint32_t mk0 = *reinterpret_cast<const uint32_t*>(blk + KV4_PARAMS_K + 8 + g * 16 + (t & 1) * 4),
                   mk1 = *reinterpret_cast<const uint32_t*>(blk + KV4_PARAMS_K + 136 + g * 16 + (t & 1) * 4);
    float score[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int r = 0; r < 4; r++) score[nt][r] = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        float part[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int r = 0; r < 4; r++) part[nt][r] = 0.0f;
        uint32_t w0 = ka_word(k0, j), w1 = ka_word(k1, j);
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
                ka_mma16(part[nt], w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u, q.b[nt][j][h][0], q.b[nt][j][h][1]);
            w0 >>= 8;
            w1 >>= 8;
        }
        const float2 a = ka_halves(j < 2 ? sk0.x : sk0.y), b = ka_halves(j < 2 ? sk1.x : sk1.y);
        const float s0 = (j & 1) ? a.y : a.x, s1 = (j & 1) ? b.y : b.x;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            score[nt][0] = fmaf(part[nt][0], s0, score[nt][0]);
            score[nt][1] = fmaf(part[nt][1], s0, score[nt][1]);
            score[nt][2] = fmaf(part[nt][2], s1, score[nt][2]);
            score[nt][3] = fmaf(part[nt][3], s1, score[nt][3]);
        }
    }
    uint32_t p[NT][2];
    bool over = false;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        float mk[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        ka_mma8(mk, mk0, mk1, q.sum[nt]);
#pragma unroll
        for (int r = 0; r < 4; r++) {
            score[nt][r] = fmaf(score[nt][r], 16777216.0f, mk[r]) * q.factor[nt][r & 1];
            if (MASKED && g + 8 * (r >> 1) >= left[nt][r & 1]) score[nt][r] = -INFINITY;
            over |= score[nt][r] > z.max[nt][r & 1] + 2.0f;
        }
    }
    if (__any_sync(S2P_FULL_MASK, over)) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                float top = fmaxf(score[nt][c], score[nt][c + 2]);
                top = fmaxf(top, __shfl_xor_sync(S2P_FULL_MASK, top, 4));
                top = fmaxf(top, __shfl_xor_sync(S2P_FULL_MASK, top, 8));
                top = fmaxf(top, __shfl_xor_sync(S2P_FULL_MASK, top, 16));
                top = fmaxf(top, z.max[nt][c]);
                const float shrink = top == -INFINITY ? 1.0f : ka_exp2(z.max[nt][c] - top);
                z.max[nt][c] = top;
                z.sum[nt][c] *= shrink;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    z.o[nt][i][c] *= shrink;
                    z.o[nt][i][c + 2] *= shrink;
                }
                z.om[nt][c] *= shrink;
                z.om[nt][c + 2] *= shrink;
            }
    }
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        float e[4];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const float top = z.max[nt][r & 1];
            e[r] = ka_exp2(score[nt][r] - (MASKED && top == -INFINITY ? 0.0f : top));
        }
        z.sum[nt][0] += e[0] + e[2];
        z.sum[nt][1] += e[1] + e[3];
        p[nt][0] = ka_transpose(ka_half2(e[0], e[1]));
        p[nt][1] = ka_transpose(ka_half2(e[2], e[3]));
    }

    const uint4 v0 = *reinterpret_cast<const uint4*>(blk + 1024 + lane * 16), v1 = *reinterpret_cast<const uint4*>(blk + 1536 + lane * 16);
    const uint4 sv0 = *reinterpret_cast<const uint4*>(blk + KV4_PARAMS_V + t * 16), sv1 = *reinterpret_cast<const uint4*>(blk + KV4_PARAMS_V + 64 + t * 16);
    uint32_t mv0 = *reinterpret_cast<const uint32_t*>(blk + KV4_PARAMS_V + 128 + t * 16 + (g & 3) * 4),
             mv1 = *reinterpret_cast<const uint32_t*>(blk + KV4_PARAMS_V + 192 + t * 16 + (g & 3) * 4);
    if (g >= 4) mv0 = mv1 = 0;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) ka_mma16(z.om[nt], mv0, 0, mv1, 0, p[nt][0], p[nt][1]);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        uint32_t w0 = j < 2 ? prmt(v0.x, v0.z, (j & 1) ? 0x7632 : 0x5410) : prmt(v0.y, v0.w, (j & 1) ? 0x7632 : 0x5410);
        uint32_t w1 = j < 2 ? prmt(v1.x, v1.z, (j & 1) ? 0x7632 : 0x5410) : prmt(v1.y, v1.w, (j & 1) ? 0x7632 : 0x5410);
        uint32_t b0[NT], b1[NT];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            b0[nt] = ka_mul2(p[nt][0], ka_word(sv0, j));
            b1[nt] = ka_mul2(p[nt][1], ka_word(sv1, j));
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
                ka_mma16(z.o[nt][2 * j + h], w0 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x000F000Fu, w1 & 0x00F000F0u, b0[nt], b1[nt]);
            w0 >>= 8;
            w1 >>= 8;
        }
    }
}

struct KaParts {
    float *max, *sum, *o; /* [slot][column](, [128]) */
    unsigned* arrived;    /* [unit] */
};

template <int NT>
__global__ void __launch_bounds__(KA_THREADS, NT == 1 ? 2 : 1)
k_kv4_attn(Kv4View cache, Kv4Rows b, const __nv_bfloat16* q, __nv_bfloat16* out, KaParts parts) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float sh_max[KA_WARPS][8 * NT], sh_sum[KA_WARPS][8 * NT];
    __shared__ long long sh_scan_ll[KA_WARPS];
    __shared__ int sh_scan[KA_WARPS], sh_last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    unsigned char* ring = smem + warp * KA_RING * KV4_BLOCK_BYTES;
    float* merge = reinterpret_cast<float*>(smem + KA_RING_BYTES);
    KaBatch batch;
    batch.upto = reinterpret_cast<long long*>(smem + KA_RING_BYTES + KA_MERGE_BYTES);
    batch.start = reinterpret_cast<int*>(batch.upto + b.n + 1);
    const int group = cache.q_heads / cache.kv_heads, rows_per = max(1, 8 * NT / group);
    const int capacity = cache.stride * S2P_B200_KV4_PAGE;

    grid_wait();
    grid_release();
    /* Rows and blocks of every entry.  Starts are made ascending and kept inside the activations, whatever row0 holds. */
    const int per = (b.n + KA_THREADS) / KA_THREADS; /* entries a thread looks at, the end of the last among them */
    {
        int top = 0;
        for (int i = 0; i < per; i++) {
            const int e = tid * per + i;
            if (e <= b.n) top = max(top, min(b.row0[e], b.rows));
        }
        int incl = top;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int o = __shfl_up_sync(S2P_FULL_MASK, incl, off);
            if (lane >= off) incl = max(incl, o);
        }
        if (lane == 31) sh_scan[warp] = incl;
        int before = __shfl_up_sync(S2P_FULL_MASK, incl, 1);
        if (lane == 0) before = 0;
        __syncthreads();
        for (int w = 0; w < warp; w++) before = max(before, sh_scan[w]);
        for (int i = 0; i < per; i++) {
            const int e = tid * per + i;
            if (e <= b.n) batch.start[e] = before = max(before, min(b.row0[e], b.rows));
        }
        __syncthreads();
    }
    auto first_of = [&](int e) { return (unsigned)b.seqs[e] < (unsigned)cache.max_seqs && b.pos0[e] <= (1 << 30) ? b.pos0[e] : -1; };
    /* positions that the row of an entry at p0 sees, its rows counted from 0 */
    auto seen_by = [&](int p0, int row) { return p0 < 0 ? 0 : (int)min((long long)p0 + row + 1, (long long)capacity); };
    auto blocks_of = [&](int e) { /* of each of the entry's units */
        return max(1, (seen_by(first_of(e), batch.start[e + 1] - batch.start[e] - 1) + 15) / 16);
    };
    {
        long long sum = 0;
        for (int i = 0; i < per; i++) {
            const int e = tid * per + i;
            if (e < b.n) {
                const int rows = batch.start[e + 1] - batch.start[e];
                sum += (long long)((rows + rows_per - 1) / rows_per) * cache.kv_heads * blocks_of(e);
            }
        }
        long long incl = sum;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const long long o = __shfl_up_sync(S2P_FULL_MASK, incl, off);
            if (lane >= off) incl += o;
        }
        if (lane == 31) sh_scan_ll[warp] = incl;
        __syncthreads();
        long long at = incl - sum;
        for (int w = 0; w < warp; w++) at += sh_scan_ll[w];
        for (int i = 0; i < per; i++) {
            const int e = tid * per + i;
            if (e <= b.n) batch.upto[e] = at;
            if (e < b.n) {
                const int rows = batch.start[e + 1] - batch.start[e];
                at += (long long)((rows + rows_per - 1) / rows_per) * cache.kv_heads * blocks_of(e);
            }
        }
        __syncthreads();
    }
    const long long total = batch.upto[b.n];
    const long long ctas = min((long long)gridDim.x, (total + KA_LEAST - 1) / KA_LEAST);
    if (blockIdx.x >= ctas) return;
    const long long begin = total * blockIdx.x / ctas, end = total * (blockIdx.x + 1) / ctas;

    int e = 0;
    { /* the last entry that begins at or before `begin` and has blocks */
        int lo = 0, hi = b.n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (batch.upto[mid] <= begin) lo = mid; else hi = mid;
        }
        e = lo;
    }
    for (long long cur = begin; cur < end;) {
        while (batch.upto[e + 1] <= cur) e++;
        const int blocks = blocks_of(e), rows = batch.start[e + 1] - batch.start[e];
        const long long inside = cur - batch.upto[e];
        const int unit = (int)(inside / blocks), x0 = (int)(inside % blocks);
        const int x1 = (int)min((long long)blocks, x0 + (end - cur));
        const int chunk = unit / cache.kv_heads, head = unit % cache.kv_heads;
        const int r0 = chunk * rows_per, n_rows = min(rows_per, rows - r0), columns = n_rows * group;
        const int row = batch.start[e] + r0, seq = b.seqs[e], p0 = first_of(e);
        const int seen = seen_by(p0, r0 + n_rows - 1), least = seen_by(p0, r0); /* by the last row and the first */
        const size_t q_stride = (size_t)cache.q_heads * 128;

        KaQuery<NT> query;
        ka_load_query<NT>(query, q + (size_t)row * q_stride + (size_t)head * group * 128, q_stride, group, columns, lane);
        KaState<NT> z;
        ka_clear(z);
        int limit[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int col = nt * 8 + 2 * t + c;
                limit[nt][c] = col < columns ? seen_by(p0, r0 + col / group) : seen;
            }

        /* this warp's blocks: x0 + warp, + KA_WARPS, ...; lane i keeps the page of the (32 n + i)-th */
        const int mine = x1 - x0 > warp ? (x1 - x0 - warp + KA_WARPS - 1) / KA_WARPS : 0;
        int page_of = -1;
        unsigned absent = 0; /* ring slots without a block */
        auto fetch = [&](int i) {
            if (i < mine) {
                if ((i & 31) == 0) {
                    const int x = x0 + warp + (i + lane) * KA_WARPS;
                    page_of = i + lane < mine && x * 16 < seen ? kv4_page(cache, seq, x * 16) : -1;
                }
                const int page = __shfl_sync(S2P_FULL_MASK, page_of, i & 31), x = x0 + warp + i * KA_WARPS;
                const unsigned bit = 1u << (i % KA_RING);
                if (page >= 0) {
                    const unsigned char* src = kv4_block(cache, page, head, x * 16) + lane * 16;
                    const uint32_t dst = smem_u32(ring + (i % KA_RING) * KV4_BLOCK_BYTES) + lane * 16;
#pragma unroll
                    for (int k = 0; k < KV4_BLOCK_BYTES / 512; k++)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + k * 512), "l"(src + k * 512) : "memory");
                    absent &= ~bit;
                } else absent |= bit;
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int i = 0; i < KA_RING - 1; i++) fetch(i);
        for (int i = 0; i < mine; i++) {
            fetch(i + KA_RING - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(KA_RING - 1) : "memory");
            __syncwarp();
            if (!(absent >> (i % KA_RING) & 1)) {
                unsigned char* blk = ring + (i % KA_RING) * KV4_BLOCK_BYTES;
                const int first = (x0 + warp + i * KA_WARPS) * 16;
                if (first + 16 <= least) {
                    const int none[NT][2] = {};
                    ka_block<NT, false>(z, query, blk, none, lane);
                } else {
                    if (first + 16 > seen) { /* nobody has written what lies behind the last position: it must not meet a zero weight as NaN */
                        const int i16 = lane & 15, at = kv4_value_param_at(i16, 0) + (lane >> 4) * 128;
                        if (first + i16 >= seen)
#pragma unroll
                            for (int j = 0; j < 4; j++) *reinterpret_cast<uint16_t*>(blk + at + 4 * j) = 0;
                        __syncwarp();
                    }
                    int left[NT][2];
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        left[nt][0] = limit[nt][0] - first;
                        left[nt][1] = limit[nt][1] - first;
                    }
                    ka_block<NT, true>(z, query, blk, left, lane);
                }
            }
            __syncwarp();
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");

        /* the warps' results together */
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                float s = z.sum[nt][c];
                s += __shfl_xor_sync(S2P_FULL_MASK, s, 4);
                s += __shfl_xor_sync(S2P_FULL_MASK, s, 8);
                s += __shfl_xor_sync(S2P_FULL_MASK, s, 16);
                if (g == 0) {
                    sh_max[warp][nt * 8 + 2 * t + c] = z.max[nt][c];
                    sh_sum[warp][nt * 8 + 2 * t + c] = s;
                }
            }
        const bool whole = x0 == 0 && x1 == blocks;
        const size_t slot = 2 * (size_t)blockIdx.x + (x0 == 0 ? 1 : 0);
        const int col = tid >> 6, dim = (tid & 63) * 2;
#pragma unroll
        for (int pass = 0; pass < 2 * NT; pass++) {
            if (pass * KA_PASS >= columns) break;
            const int nt = pass >> 1;
#pragma unroll
            for (int c = 0; c < 2; c++) {
                float* to = merge + ((warp * KA_PASS) + 2 * (t & 1) + c) * 128 + 4 * g;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float m = __shfl_sync(S2P_FULL_MASK, z.om[nt][c], 4 * j + t);
                    if ((t >> 1) == (pass & 1))
                        *reinterpret_cast<float4*>(to + 32 * j) =
                            make_float4(fmaf(z.o[nt][2 * j][c], 16777216.0f, m), fmaf(z.o[nt][2 * j][c + 2], 1048576.0f, m),
                                        fmaf(z.o[nt][2 * j + 1][c], 16777216.0f, m), fmaf(z.o[nt][2 * j + 1][c + 2], 1048576.0f, m));
                }
            }
            __syncthreads();
            const int at = pass * KA_PASS + col;
            if (at < columns) {
                float top = -INFINITY, sum = 0.0f, a0 = 0.0f, a1 = 0.0f;
#pragma unroll
                for (int w = 0; w < KA_WARPS; w++) top = fmaxf(top, sh_max[w][at]);
#pragma unroll
                for (int w = 0; w < KA_WARPS; w++) {
                    const float scale = sh_max[w][at] == -INFINITY && sh_sum[w][at] == 0.0f ? 0.0f : ka_exp2(sh_max[w][at] - (top == -INFINITY ? 0.0f : top));
                    const float2 v = *reinterpret_cast<const float2*>(merge + (w * KA_PASS + col) * 128 + dim);
                    sum = fmaf(sh_sum[w][at], scale, sum);
                    a0 = fmaf(v.x, scale, a0);
                    a1 = fmaf(v.y, scale, a1);
                }
                if (whole) {
                    const float r = sum == 0.0f ? 0.0f : 1.0f / sum;
                    const __nv_bfloat162 y = __floats2bfloat162_rn(a0 * r, a1 * r);
                    *reinterpret_cast<__nv_bfloat162*>(out + (size_t)(row + at / group) * q_stride + (size_t)(head * group + at % group) * 128 + dim) = y;
                } else {
                    if ((tid & 63) == 0) {
                        parts.max[slot * KV4_PART_COLS + at] = top;
                        parts.sum[slot * KV4_PART_COLS + at] = sum;
                    }
                    *reinterpret_cast<float2*>(parts.o + (slot * KV4_PART_COLS + at) * 128 + dim) = make_float2(a0, a1);
                }
            }
            __syncthreads();
        }
        if (!whole) {
            /* CTA of block x of the line: the largest c with total c / ctas <= x */
            const long long u0 = batch.upto[e] + (long long)unit * blocks, u1 = u0 + blocks - 1;
            const int c0 = (int)(((u0 + 1) * ctas - 1) / total), c1 = (int)(((u1 + 1) * ctas - 1) / total);
            if (tid == 0) {
                /* the row's first column stands for the unit: rows of units are distinct */
                unsigned* arrived = parts.arrived + (size_t)row * cache.kv_heads + head;
                __threadfence();
                const unsigned old = atomicAdd(arrived, 1u);
                sh_last = old == (unsigned)(c1 - c0);
                if (sh_last) *arrived = 0;
                __threadfence();
            }
            __syncthreads();
            if (sh_last) {
                for (int at = col; at < columns; at += KA_PASS) {
                    float top = -INFINITY, sum = 0.0f, a0 = 0.0f, a1 = 0.0f;
                    for (int c = c0; c <= c1; c++) {
                        const size_t s = 2 * (size_t)c + (total * c / ctas <= u0 ? 1 : 0);
                        top = fmaxf(top, __ldcg(parts.max + s * KV4_PART_COLS + at));
                    }
                    for (int c = c0; c <= c1; c++) {
                        const size_t s = (2 * (size_t)c + (total * c / ctas <= u0 ? 1 : 0)) * KV4_PART_COLS + at;
                        const float m = __ldcg(parts.max + s), l = __ldcg(parts.sum + s);
                        const float2 v = __ldcg(reinterpret_cast<const float2*>(parts.o + s * 128 + dim));
                        const float scale = m == -INFINITY && l == 0.0f ? 0.0f : ka_exp2(m - (top == -INFINITY ? 0.0f : top));
                        sum = fmaf(l, scale, sum);
                        a0 = fmaf(v.x, scale, a0);
                        a1 = fmaf(v.y, scale, a1);
                    }
                    const float r = sum == 0.0f ? 0.0f : 1.0f / sum;
                    const __nv_bfloat162 y = __floats2bfloat162_rn(a0 * r, a1 * r);
                    *reinterpret_cast<__nv_bfloat162*>(out + (size_t)(row + at / group) * q_stride + (size_t)(head * group + at % group) * 128 + dim) = y;
                }
            }
            __syncthreads();
        }
        cur += x1 - x0;
    }
}

extern "C" size_t kv4_counter_bytes(int rows, int kv_heads) { return ((size_t)rows * (size_t)kv_heads * sizeof(unsigned) + 255) / 256 * 256; }

template <int NT>
static cudaError_t launch_attn(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int layer, const void* q, void* out, cudaStream_t st) {
    const size_t smem = KA_RING_BYTES + KA_MERGE_BYTES + ka_batch_bytes(b->n);
    static bool attr_set[64] = {false};
    static int sms[64] = {0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!attr_set[dev]) {
        e = cudaFuncSetAttribute(k_kv4_attn<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)(KA_RING_BYTES + KA_MERGE_BYTES + ka_batch_bytes(S2P_B200_KV4_MAX_BATCH)));
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev);
        if (e != cudaSuccess) return e;
        attr_set[dev] = true;
    }
    KaParts p;
    unsigned char* at = static_cast<unsigned char*>(c->work) + KV4_STATUS_BYTES;
    p.arrived = reinterpret_cast<unsigned*>(at);
    at += kv4_counter_bytes(b->rows, c->kv_heads);
    p.o = reinterpret_cast<float*>(at);
    p.max = p.o + (size_t)2 * KV4_MAX_CTAS * KV4_PART_COLS * 128;
    p.sum = p.max + (size_t)2 * KV4_MAX_CTAS * KV4_PART_COLS;
    const int grid = sms[dev] * (NT == 1 ? 2 : 1);
    return launch_after(k_kv4_attn<NT>, dim3((unsigned)(grid < KV4_MAX_CTAS ? grid : KV4_MAX_CTAS)), KA_THREADS, smem, st, kv4_view(*c, layer), kv4_rows(*b),
                        static_cast<const __nv_bfloat16*>(q), static_cast<__nv_bfloat16*>(out), p);
}

extern "C" cudaError_t kv4_attention(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int layer, const void* q, void* out, cudaStream_t st) {
    const int group = c->q_heads / c->kv_heads, rows = b->max_rows > 1 ? b->max_rows : 1;
    return rows * group <= 8 ? launch_attn<1>(c, b, layer, q, out, st) : launch_attn<2>(c, b, layer, q, out, st);
}

}  // namespace s2p
