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
 *            block normally costs one vote.  The maximum is taken off before a score is scaled: the scaled one would be rounded, by thousands where queries are
 *            large enough, and what is left of the largest score would then be an exponent that no f16 has.  p is rounded to f16, 11 bits, for the products.
 *   values   O^T [128 channels x columns]: A = values, the pairs of positions put together by byte permutation, B = p^T, which is
 *            S^T transposed in registers (movmatrix), times s of the group, rounded to f16 once more.  Weights (at most 4) are lifted by a power of two, 2^12 to begin with, so that the
 *            product has all of f16's bits down to s = 2^-17 for a weight of 2^-9: without it values of 1e-4 came out 1% off at 16000 positions, of 1e-5 67%.  Where an s is
 *            met that would take the product to 2^15, the lift goes down and what has been summed with it, as for a new maximum.
 *
 * The cache is read once, so what bounds single tokens is HBM.  A CTA or a warp takes an equal part of a unit, or an equal stretch of the
 * line of all units' blocks; a warp walks its blocks through a ring of asynchronous copies of its own.  A unit that several share is put
 * together by the last of them to arrive, in their order, so that the result does not depend on timing. */
#include <limits.h>
#include "kv4.cuh"
#include "pipe.cuh"

namespace s2p {

constexpr int KA_WARPS = 8, KA_THREADS = KA_WARPS * 32, KA_PIECE = 4, KA_STAGES = 2; /* blocks that a warp asks for at a time (of one page), and such pieces in its ring */
constexpr int KA_RING_BYTES = KA_WARPS * KA_STAGES * KA_PIECE * KV4_BLOCK_BYTES;
constexpr int KA_PASS = 4;                                         /* columns merged at a time */
constexpr int KA_MERGE_BYTES = KA_WARPS * KA_PASS * 128 * 4;
constexpr int KA_LEAST_CTA = KA_WARPS, KA_LEAST_WARP = 8;          /* blocks that make a worker worth its while */
/* (Row, head) columns of a kv head up to which an entry is this kernel's rather than that of the tensor cores: alone, and next to longer slices, where
 * most bring a token.  us here and there, 32 query and 8 kv heads (8 and 8 the same by columns), 32, 36, 48, 64 columns:
 *   one sequence of  500     12.0 12.0 12.1 12.1 and 16.8 16.9 16.9 17.2      16 of 1000  27 30 31 36 and 34 35 35 35
 *                   1100     18.7 16.8 17.0 18.4 and 18.1 18.2 18.3 18.7      16 of 4000  62 73 73 97 and 78 82 82 82
 *                   8000     21.9 24.2 24.3 27.6 and 25.4 25.5 25.5 26.9      64 of 300   22 46 46 53 and -- 68 68 69
 *                  20000     29.1 72.2 76.6 68.9 and   --  36.6 36.5 38.0
 * The crossing goes by the context, which the host does not know: 64 is the better side for short and medium ones, and costs up to twice the time for one long sequence. */
constexpr int KA_FEW = 64, KA_FEW_BESIDE = 32;
/* How the work is cut (us, 32 query and 8 kv heads, one row a sequence).  Units each cut into equal parts, one to a CTA, its warps joined through shared memory,
 * wherever there are no more units than CTAs: 15 sequences of 1500 13.3, by warps below 20.6; up to KA_LONG blocks to a warp, where the warps' barriers cost more
 * than the partials that they save (9 of 8000 28.2 and 27.5, 12 of 4000 24.0 and 22.8), and where no part has KA_SECOND blocks more than an equal share (one
 * sequence of 2000 among 15 of 1000, 67 more: 14.6 and 16.4; of 3000, 130 more: 18.2 and 17.8).  Units of up to KA_WHOLE blocks are not cut even so, since putting
 * parts together takes longer than more blocks do (one sequence of 512 whole 7.8, cut 9.0; 8 of 1000 11.0 and 12.0, of 1250 11.7 and 12.0; one of 1000 9.9 and 9.6, of
 * 1100 10.9 and 9.7).  Otherwise a warp is a worker by itself and leaves a partial.
 * Equal parts of each unit again (64 of 512: 18.0, 24 of 2500: 23.5), unless a part has KA_SECOND_WARP blocks more than an equal stretch of the line of all units'
 * blocks, in which many warps end one unit and begin the next (64 of 512 20.5, 24 of 2500 26.2; but 32 of 8192, 18 more: 58.5, in parts 66).  (Taken before weights were
 * lifted, which adds 1 to 2% on either side.) */
constexpr int KA_SECOND = 120, KA_SECOND_WARP = 8, KA_LONG = 20, KA_WHOLE = 64;

struct KaBatch { /* in shared memory, [n (+ 1)] */
    unsigned* upto;  /* blocks of all units before entry e */
    int* start;      /* its first row */
    int* first;      /* its first position, or -1 */
    int* seq;
};
__host__ __device__ static inline size_t ka_batch_bytes(int n) { return (size_t)(n + 1) * 16; }
__device__ __forceinline__ KaBatch ka_batch(unsigned char* at, int n) {
    KaBatch s;
    s.upto = reinterpret_cast<unsigned*>(at);
    s.start = reinterpret_cast<int*>(s.upto + n + 1);
    s.first = s.start + n + 1;
    s.seq = s.first + n + 1;
    return s;
}

__device__ __forceinline__ void ka_mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
/* the same onto zeros, without registers set to zero first */
__device__ __forceinline__ void ka_mma16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void ka_mma8_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5}, {%6}, {%7, %7, %7, %7};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(b0), "f"(0.0f));
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
    float factor[NT][2];     /* of the lane's two score columns: from scores over 2^24 to base-2 logits */
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
        const float f = down * (16777216.0f * 1.4426950408889634f * 0.08838834764831845f); /* 2^24 log2(e) / sqrt(128) */
        z.factor[nt][0] = __shfl_sync(S2P_FULL_MASK, f, 8 * t);
        z.factor[nt][1] = __shfl_sync(S2P_FULL_MASK, f, 8 * t + 4);
    }
}

template <int NT> struct KaState {
    float o[NT][8][4]; /* [column tile][channel tile 2 j + h]: rows 4 g + 2 h (16 times 2^-24 that of the second) and + 1 of group j */
    float om[NT][4];   /* [0], [1], in lanes with g < 4: sum of p m of group g; [2], [3]: sum of p */
    float max[NT][2]; /* of the scores before they are scaled */
    float lift;       /* weights are 2^((score - max) factor + lift) */
    uint32_t watch;   /* in both halves: 0x8000 less the f16 that s has to stay below, 2^(13 - lift) */
};
constexpr float KA_LIFT = 12.0f;
constexpr uint32_t KA_WATCH = 0x40004000u; /* s < 2 */
constexpr float KA_NONE = -1e38f; /* maximum of a column that has seen nothing: finite, so that weights relative to it are zero */
template <int NT> __device__ __forceinline__ void ka_clear(KaState<NT>& z) {
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) z.o[nt][i][r] = 0.0f;
#pragma unroll
        for (int r = 0; r < 4; r++) z.om[nt][r] = 0.0f;
        z.max[nt][0] = z.max[nt][1] = KA_NONE;
    }
    z.lift = KA_LIFT;
    z.watch = KA_WATCH;
}

/* what a column's sums are relative to, for those who put parts together */
template <int NT> __device__ __forceinline__ float ka_base(const KaState<NT>& z, const KaQuery<NT>& q, int nt, int c) {
    return z.max[nt][c] == KA_NONE ? -INFINITY : fmaf(z.max[nt][c], q.factor[nt][c], -z.lift);
}

/* Two blocks of 16 positions from shared memory: their instructions interleave.  Where `masked`, left(column tile, 0 or 1) says how many of the 32
 * positions the lane's first or second column of the tile sees.  (There is one copy of this code, for the instruction cache: one token at a
 * short context runs it once, and a second copy for whole blocks cost more there than the test does.) */
template <int NT, class Left>
__device__ __forceinline__ void ka_blocks(KaState<NT>& z, const KaQuery<NT>& q, const unsigned char* const (&blk)[2], bool masked, Left left, int lane) {
    constexpr int NB = 2;
    const int g = lane >> 2, t = lane & 3;
    float score[NB][NT][4];
#pragma unroll
    for (int n = 0; n < NB; n++) {
        const uint4 k0 = *reinterpret_cast<const uint4*>(blk[n] + lane * 16), k1 = *reinterpret_cast<const uint4*>(blk[n] + 512 + lane * 16);
        const uint2 sk0 = *reinterpret_cast<const uint2*>(blk[n] + KV4_PARAMS_K + g * 16), sk1 = *reinterpret_cast<const uint2*>(blk[n] + KV4_PARAMS_K + 128 + g * 16);
        const uint32_t mk0 = *reinterpret_cast<const uint32_t*>(blk[n] + KV4_PARAMS_K + 8 + g * 16 + (t & 1) * 4),
                       mk1 = *reinterpret_cast<const uint32_t*>(blk[n] + KV4_PARAMS_K + 136 + g * 16 + (t & 1) * 4);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float part[NT][4];
            uint32_t w0 = ka_word(k0, j), w1 = ka_word(k1, j);
#pragma unroll
            for (int h = 0; h < 2; h++) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
                    if (h == 0) ka_mma16_first(part[nt], w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u, q.b[nt][j][h][0], q.b[nt][j][h][1]);
                    else ka_mma16(part[nt], w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u, q.b[nt][j][h][0], q.b[nt][j][h][1]);
                w0 >>= 8;
                w1 >>= 8;
            }
            const float2 a = ka_halves(j < 2 ? sk0.x : sk0.y), b = ka_halves(j < 2 ? sk1.x : sk1.y);
            const float s0 = (j & 1) ? a.y : a.x, s1 = (j & 1) ? b.y : b.x;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int r = 0; r < 4; r++) score[n][nt][r] = j ? fmaf(part[nt][r], r < 2 ? s0 : s1, score[n][nt][r]) : part[nt][r] * (r < 2 ? s0 : s1);
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float mk[4];
            ka_mma8_first(mk, mk0, mk1, q.sum[nt]);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                score[n][nt][r] = fmaf(mk[r], 5.9604645e-8f, score[n][nt][r]); /* 2^-24, like the codes */
            }
        }
    }
    if (masked) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int see = left(nt, c) - g;
#pragma unroll
                for (int n = 0; n < NB; n++) {
                    if (16 * n >= see) score[n][nt][c] = -INFINITY;
                    if (16 * n + 8 >= see) score[n][nt][c + 2] = -INFINITY;
                }
            }
    }
    /* the s of a block's values are 128 bytes: a word a lane */
    const uint32_t vs0 = *reinterpret_cast<const uint32_t*>(blk[0] + KV4_PARAMS_V + 4 * lane), vs1 = *reinterpret_cast<const uint32_t*>(blk[1] + KV4_PARAMS_V + 4 * lane);
    bool over = (((vs0 + z.watch) | (vs1 + z.watch)) & 0x80008000u) != 0;
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
            float top = fmaxf(score[0][nt][c], score[0][nt][c + 2]);
#pragma unroll
            for (int n = 1; n < NB; n++) top = fmaxf(top, fmaxf(score[n][nt][c], score[n][nt][c + 2]));
            over |= (top - z.max[nt][c]) * q.factor[nt][c] > 2.0f;
        }
    if (__any_sync(S2P_FULL_MASK, over)) {
        const uint32_t s2 = __vmaxu2(vs0, vs1), s1 = __reduce_max_sync(S2P_FULL_MASK, max(s2 & 0xFFFFu, s2 >> 16));
        const float was = z.lift;
        if (s1 + (z.watch & 0xFFFFu) >= 0x8000u) {
            const uint32_t below = ((s1 >> 10) + 1) << 10; /* the next power of two above s1, as an f16: 2^(below / 2^10 - 15) */
            z.watch = (0x8000u - below) * 0x10001u;
            z.lift = 28.0f - (float)(below >> 10);
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                float top = fmaxf(score[0][nt][c], score[0][nt][c + 2]);
#pragma unroll
                for (int n = 1; n < NB; n++) top = fmaxf(top, fmaxf(score[n][nt][c], score[n][nt][c + 2]));
                top = fmaxf(top, __shfl_xor_sync(S2P_FULL_MASK, top, 4));
                top = fmaxf(top, __shfl_xor_sync(S2P_FULL_MASK, top, 8));
                top = fmaxf(top, __shfl_xor_sync(S2P_FULL_MASK, top, 16));
                top = fmaxf(top, z.max[nt][c]);
                const float shrink = ka_exp2(fmaf(z.max[nt][c] - top, q.factor[nt][c], z.lift - was));
                z.max[nt][c] = top;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    z.o[nt][i][c] *= shrink;
                    z.o[nt][i][c + 2] *= shrink;
                }
                z.om[nt][c] *= shrink;
                z.om[nt][c + 2] *= shrink;
            }
    }
    uint32_t p[NB][NT][2];
#pragma unroll
    for (int n = 0; n < NB; n++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float e[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                e[r] = ka_exp2(fmaf(score[n][nt][r] - z.max[nt][r & 1], q.factor[nt][r & 1], z.lift));
            }
            p[n][nt][0] = ka_transpose(ka_half2(e[0], e[1]));
            p[n][nt][1] = ka_transpose(ka_half2(e[2], e[3]));
        }
#pragma unroll
    for (int n = 0; n < NB; n++) {
        const uint4 v0 = *reinterpret_cast<const uint4*>(blk[n] + 1024 + lane * 16), v1 = *reinterpret_cast<const uint4*>(blk[n] + 1536 + lane * 16);
        const uint4 sv0 = *reinterpret_cast<const uint4*>(blk[n] + KV4_PARAMS_V + t * 16), sv1 = *reinterpret_cast<const uint4*>(blk[n] + KV4_PARAMS_V + 64 + t * 16);
        const uint32_t mv0 = *reinterpret_cast<const uint32_t*>(blk[n] + KV4_PARAMS_V + 128 + t * 16 + (g & 3) * 4),
                       mv1 = *reinterpret_cast<const uint32_t*>(blk[n] + KV4_PARAMS_V + 192 + t * 16 + (g & 3) * 4);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) ka_mma16(z.om[nt], mv0, 0x3C003C00u, mv1, 0x3C003C00u, p[n][nt][0], p[n][nt][1]); /* the lower rows: ones */
#pragma unroll
        for (int j = 0; j < 4; j++) {
            uint32_t w0 = j < 2 ? prmt(v0.x, v0.z, (j & 1) ? 0x7632 : 0x5410) : prmt(v0.y, v0.w, (j & 1) ? 0x7632 : 0x5410);
            uint32_t w1 = j < 2 ? prmt(v1.x, v1.z, (j & 1) ? 0x7632 : 0x5410) : prmt(v1.y, v1.w, (j & 1) ? 0x7632 : 0x5410);
            uint32_t b0[NT], b1[NT];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                b0[nt] = ka_mul2(p[n][nt][0], ka_word(sv0, j));
                b1[nt] = ka_mul2(p[n][nt][1], ka_word(sv1, j));
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
}

/* Partial results: slot 2 w + 1 where worker w begins a unit that others end, 2 w where it goes on with one. */
static_assert((size_t)KV4_PARTS * (128 + 2) * sizeof(float) <= KV4_AREA_BYTES, "the tokens' partials");
struct KaParts {
    float *max, *sum, *o; /* [slot][8 NT columns](, [128]); max: ka_base */
    unsigned* arrived;    /* [row][kv head] of a unit's first row */
};

/* What the workers from, from + step, ... up to `last` left of a unit (starts: the one that begins it), for columns base .. base + 3: running
 * maximum, sum, and channels 4 lane .. 4 lane + 3 of the weighted values.  Sixteen loads are under way at a time. */
template <int COLS>
__device__ __forceinline__ void ka_gather(const KaParts& parts, int starts, int from, int step, int last, int base, int columns, int lane, float (&top)[KA_PASS],
                                          float (&sum)[KA_PASS], float4 (&acc)[KA_PASS]) {
#pragma unroll
    for (int k = 0; k < KA_PASS; k++) {
        top[k] = -INFINITY;
        sum[k] = 0.0f;
        acc[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    for (int w0 = from; w0 <= last; w0 += 4 * step) {
        float4 v[4][KA_PASS];
        float m[4][KA_PASS], l[4][KA_PASS];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int w = w0 + i * step;
            const size_t at = (size_t)(2 * w + (w == starts)) * COLS + base;
#pragma unroll
            for (int k = 0; k < KA_PASS; k++) {
                const bool there = w <= last && base + k < columns;
                m[i][k] = there ? __ldcg(parts.max + at + k) : -INFINITY;
                l[i][k] = there ? __ldcg(parts.sum + at + k) : 0.0f;
                v[i][k] = there ? __ldcg(reinterpret_cast<const float4*>(parts.o + (at + k) * 128) + lane) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
        }
#pragma unroll
        for (int k = 0; k < KA_PASS; k++) {
            const float now = fmaxf(fmaxf(fmaxf(m[0][k], m[1][k]), fmaxf(m[2][k], m[3][k])), top[k]);
            const float base2 = now == -INFINITY ? 0.0f : now, keep = ka_exp2(top[k] - base2);
            sum[k] *= keep;
            acc[k].x *= keep; acc[k].y *= keep; acc[k].z *= keep; acc[k].w *= keep;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float scale = ka_exp2(m[i][k] - base2);
                sum[k] = fmaf(l[i][k], scale, sum[k]);
                acc[k].x = fmaf(v[i][k].x, scale, acc[k].x);
                acc[k].y = fmaf(v[i][k].y, scale, acc[k].y);
                acc[k].z = fmaf(v[i][k].z, scale, acc[k].z);
                acc[k].w = fmaf(v[i][k].w, scale, acc[k].w);
            }
            top[k] = now;
        }
    }
}

__device__ __forceinline__ void ka_store(__nv_bfloat16* to, float4 v, float sum) {
    const float r = sum == 0.0f ? 0.0f : 1.0f / sum;
    const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x * r, v.y * r), hi = __floats2bfloat162_rn(v.z * r, v.w * r);
    *reinterpret_cast<uint2*>(to) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}

template <int NT>
__global__ void __launch_bounds__(KA_THREADS, 1)
k_kv4_attn(Kv4View cache, Kv4Rows b, int few, int group, int rows_per, const __nv_bfloat16* q, __nv_bfloat16* out, KaParts parts) {
    constexpr int COLS = 8 * NT;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float sh_max[KA_WARPS][COLS], sh_sum[KA_WARPS][COLS];
    __shared__ struct { unsigned by_warp, cut, workers, share, more; } sh_line;
    __shared__ int sh_last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    unsigned char* ring = smem + warp * KA_STAGES * KA_PIECE * KV4_BLOCK_BYTES;
    float* merge = reinterpret_cast<float*>(smem + KA_RING_BYTES);
    const KaBatch batch = ka_batch(smem + KA_RING_BYTES + KA_MERGE_BYTES, b.n);
    const int capacity = cache.stride * S2P_B200_KV4_PAGE;

    grid_wait();
    grid_release();
    /* Rows and blocks of every entry.  Starts are made ascending and kept inside the activations, whatever row0 holds. */
    auto seen_by = [&](int p0, int row) { /* positions that a row of an entry at p0 sees, its rows counted from 0 */
        return p0 < 0 ? 0 : (int)min((long long)p0 + row + 1, (long long)capacity);
    };
    auto blocks_of = [&](int e) { /* of each of the entry's units */
        return max(1, (seen_by(batch.first[e], batch.start[e + 1] - batch.start[e] - 1) + 15) / 16);
    };
    auto units_of = [&](int e) { /* entries of more rows than `few` are another kernel's */
        const int rows = batch.start[e + 1] - batch.start[e];
        return rows > few || !rows ? 0 : rows <= rows_per ? cache.kv_heads : (rows + rows_per - 1) / rows_per * cache.kv_heads;
    };
    /* Brought by all, worked out by one warp, 128 entries at a time: two barriers.  (By all warps, with a barrier for every sum, 0.6 us more.) */
    for (int e = tid; e <= b.n; e += KA_THREADS) {
        const int r = b.row0[e];
        if (e < b.n) {
            const int seq = b.seqs[e], p0 = b.pos0[e];
            batch.seq[e] = seq;
            batch.first[e] = (unsigned)seq < (unsigned)cache.max_seqs && p0 <= (1 << 30) ? p0 : -1;
        }
        batch.start[e] = min(r, b.rows);
    }
    __syncthreads();
    auto before = [&](unsigned v, unsigned& carry) { /* carry + the lanes before this one; carry goes on */
        unsigned at = v;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const unsigned o = __shfl_up_sync(S2P_FULL_MASK, at, off);
            if (lane >= off) at += o;
        }
        const unsigned mine = carry + at - v;
        carry += __shfl_sync(S2P_FULL_MASK, at, 31);
        return mine;
    };
    if (warp == 0) {
        int top = 0;
        for (int e0 = 0; e0 <= b.n; e0 += 128) {
            int r[4], run = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int e = e0 + 4 * lane + i;
                if (e <= b.n) run = max(run, batch.start[e]);
                r[i] = run;
            }
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int o = __shfl_up_sync(S2P_FULL_MASK, run, off);
                if (lane >= off) run = max(run, o);
            }
            const int left = __shfl_up_sync(S2P_FULL_MASK, run, 1), base = max(top, lane ? left : 0);
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (e0 + 4 * lane + i <= b.n) batch.start[e0 + 4 * lane + i] = max(r[i], base);
            top = max(top, __shfl_sync(S2P_FULL_MASK, run, 31));
        }
        __syncwarp();
        /* upto[e] = the blocks of the entries before e */
        unsigned units = 0, total = 0, most = 0;
        for (int e0 = 0; e0 <= b.n; e0 += 128) {
            unsigned v[4], sum = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int e = e0 + 4 * lane + i;
                const unsigned u = e < b.n ? (unsigned)units_of(e) : 0u, l = u ? (unsigned)blocks_of(e) : 0u;
                units += u;
                most = max(most, l);
                v[i] = u * l;
                sum += v[i];
            }
            unsigned at = before(sum, total);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int e = e0 + 4 * lane + i;
                if (e <= b.n) batch.upto[e] = at;
                at += v[i];
            }
        }
        units = __reduce_add_sync(S2P_FULL_MASK, units);
        most = __reduce_max_sync(S2P_FULL_MASK, most);
        const unsigned grid = gridDim.x, warps = grid * KA_WARPS;
        /* parts of at most this many blocks are no more than there are workers; the longest of those parts */
        auto cut_for = [&](unsigned workers, unsigned least) { return max(least, (total + workers - units - 1) / (workers - units)); };
        auto part_of = [&](unsigned cut) { return cut ? (most + (most + cut - 1) / cut - 1) / max(1u, (most + cut - 1) / cut) : 0u; };
        unsigned cut = units < grid && total < warps * KA_LONG ? most <= KA_WHOLE ? max(most, 1u) : cut_for(grid, KA_LEAST_CTA) : 0;
        bool by_warp = !cut || part_of(cut) > total / grid + KA_SECOND;
        if (by_warp) {
            cut = units < warps ? cut_for(warps, KA_LEAST_WARP) : 0;
            if (part_of(cut) > total / warps + KA_SECOND_WARP) cut = 0;
        }
        if (lane == 0) {
            const unsigned workers = min(warps, (total + KA_LEAST_WARP - 1) / KA_LEAST_WARP);
            sh_line.by_warp = by_warp;
            sh_line.cut = cut;
            /* worker w of the line has `share` blocks, the first `more` workers one more */
            sh_line.workers = workers;
            sh_line.share = workers ? total / workers : 1;
            sh_line.more = workers ? total - sh_line.share * workers : 0;
        }
    }
    __syncthreads();
    const bool by_warp = sh_line.by_warp;
    const unsigned share = sh_line.share, more = sh_line.more, worker = by_warp ? warp * gridDim.x + blockIdx.x : blockIdx.x;
    unsigned begin = 0, end = 0;
    int e = 0, w_first = -1, w_last = -1; /* the entry; of a unit in parts: its workers */
    if (const unsigned longest = sh_line.cut) {
        unsigned carry = 0;
        for (int e0 = 0; e0 < b.n && carry <= worker; e0 += 32) {
            const int mine = e0 + lane;
            const unsigned u = mine < b.n ? (unsigned)units_of(mine) : 0u, l = u ? (unsigned)blocks_of(mine) : 0u, cuts = (l + longest - 1) / longest;
            const unsigned at = before(u * cuts, carry), found = __ballot_sync(S2P_FULL_MASK, worker >= at && worker - at < u * cuts);
            if (found) {
                const int who = __ffs(found) - 1;
                const unsigned in = worker - __shfl_sync(S2P_FULL_MASK, at, who), n = __shfl_sync(S2P_FULL_MASK, cuts, who), blocks = __shfl_sync(S2P_FULL_MASK, l, who);
                const unsigned unit = in / n, c = in - unit * n, piece = blocks / n, rest = blocks - piece * n;
                e = e0 + who;
                begin = batch.upto[e] + unit * blocks + piece * c + min(c, rest);
                end = begin + piece + (c < rest);
                w_first = (int)(worker - c);
                w_last = w_first + (int)n - 1;
            }
        }
    } else if (worker < sh_line.workers) {
        begin = share * worker + min(worker, more);
        end = begin + share + (worker < more);
        int lo = 0, hi = b.n;
        while (hi - lo > 1) { /* the last entry that begins at or before `begin` */
            const int mid = (lo + hi) >> 1;
            if (batch.upto[mid] <= begin) lo = mid; else hi = mid;
        }
        e = lo;
    }
    if (begin == end) return;
    auto worker_of = [&](unsigned x) { return x < (share + 1) * more ? x / (share + 1) : more + (x - (share + 1) * more) / share; };

    struct Segment { /* the stretch's part in one unit */
        int row, n_rows, r0, head, seq, p0, seen, least, blocks, x0, x1, w0, w1; /* blocks x0 .. x1 - 1 of `blocks`; the workers of the unit */
        int xa, xb, pieces;                                                    /* this warp's blocks, in pieces that end where a page does */
    };
    auto segment = [&](unsigned cur) {
        Segment s;
        while (batch.upto[e + 1] <= cur) e++; /* entries without rows */
        const int rows = batch.start[e + 1] - batch.start[e];
        s.blocks = blocks_of(e);
        const unsigned inside = cur - batch.upto[e];
        const unsigned unit = inside / (unsigned)s.blocks;
        s.x0 = (int)(inside - unit * (unsigned)s.blocks);
        s.x1 = s.x0 + (int)min((unsigned)(s.blocks - s.x0), end - cur);
        s.w0 = w_first >= 0 ? w_first : (int)worker_of(cur - (unsigned)s.x0);
        s.w1 = w_first >= 0 ? w_last : (int)worker_of(cur - (unsigned)s.x0 + (unsigned)s.blocks - 1);
        s.xa = s.x0;
        s.xb = s.x1;
        if (!by_warp) {
            const int each = (s.x1 - s.x0) / KA_WARPS, over = (s.x1 - s.x0) % KA_WARPS;
            s.xa = s.x0 + each * warp + min(warp, over);
            s.xb = s.xa + each + (warp < over);
        }
        s.pieces = s.xb > s.xa ? (s.xb - 1) / KA_PIECE - s.xa / KA_PIECE + 1 : 0;
        const int chunk = (int)(unit / (unsigned)cache.kv_heads);
        s.head = (int)unit - chunk * cache.kv_heads;
        s.r0 = chunk * rows_per;
        s.n_rows = min(rows_per, rows - s.r0);
        s.row = batch.start[e] + s.r0;
        s.seq = batch.seq[e];
        s.p0 = batch.first[e];
        s.seen = seen_by(s.p0, s.r0 + s.n_rows - 1); /* by the last row */
        s.least = seen_by(s.p0, s.r0);               /* ... and the first */
        return s;
    };
    int page_of = -1;    /* lane i keeps the page of the (32 n + i)-th piece */
    unsigned absent = 0; /* stages without a page */
    auto fetch = [&](const Segment& s, int i) {
        if (i < s.pieces) {
            const int at = s.xa / KA_PIECE + i;
            if ((i & 31) == 0) page_of = i + lane < s.pieces ? kv4_page(cache, s.seq, (at + lane) * KA_PIECE * 16) : -1;
            const int page = __shfl_sync(S2P_FULL_MASK, page_of, i & 31);
            const int from = max(s.xa, KA_PIECE * at), n = min(min(s.xb, KA_PIECE * (at + 1)), (s.seen + 15) / 16) - from; /* (an entry that sees nothing has a block, too) */
            const unsigned bit = 1u << (i % KA_STAGES);
            if (page >= 0 && n > 0) {
                const unsigned char* src = kv4_block(cache, page, s.head, from * 16) + lane * 16;
                uint32_t dst = smem_u32(ring) + (i % KA_STAGES) * KA_PIECE * KV4_BLOCK_BYTES + lane * 16;
                for (int x = 0; x < n; x++, src += KV4_BLOCK_BYTES, dst += KV4_BLOCK_BYTES)
#pragma unroll
                    for (int k = 0; k < KV4_BLOCK_BYTES / 512; k++)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + k * 512), "l"(src + k * 512) : "memory");
                absent &= ~bit;
            } else absent |= bit;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };

    const size_t q_stride = (size_t)cache.q_heads * 128;
    unsigned cur = begin;
    Segment s = segment(cur);
#pragma unroll
    for (int i = 0; i < KA_STAGES - 1; i++) fetch(s, i);
    for (;;) {
        const int columns = s.n_rows * group, row = s.row, head = s.head, r0 = s.r0, p0 = s.p0, seen = s.seen;
        KaQuery<NT> query;
        ka_load_query<NT>(query, q + (size_t)row * q_stride + (size_t)head * group * 128, q_stride, group, columns, lane);
        KaState<NT> z;
        ka_clear(z);
        for (int i = 0; i < s.pieces; i++) {
            fetch(s, i + KA_STAGES - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(KA_STAGES - 1) : "memory");
            __syncwarp();
            if (!(absent >> (i % KA_STAGES) & 1)) {
                unsigned char* blk = ring + (i % KA_STAGES) * KA_PIECE * KV4_BLOCK_BYTES;
                int x = max(s.xa, KA_PIECE * (s.xa / KA_PIECE + i));
                const int to = min(min(s.xb, KA_PIECE * (s.xa / KA_PIECE + i + 1)), (seen + 15) / 16), plain = min(to, s.least / 16); /* blocks that every row sees whole */
                for (; x < to; x += 2, blk += 2 * KV4_BLOCK_BYTES) {
                    const int first = x * 16;
                    if (first + 32 > seen) { /* nobody has written what lies behind the last position: it must not meet a zero weight as NaN */
                        const int behind = first + lane;
                        unsigned char* at = blk + (lane >> 4) * KV4_BLOCK_BYTES + kv4_value_param_at(lane & 15, 0);
                        if (behind >= seen && x + (lane >> 4) < to)
#pragma unroll
                            for (int j = 0; j < 4; j++) *reinterpret_cast<uint16_t*>(at + 4 * j) = *reinterpret_cast<uint16_t*>(at + 128 + 4 * j) = 0;
                        __syncwarp();
                    }
                    /* an odd last block comes twice, the second time behind everybody's sight */
                    const unsigned char* const two[2] = {blk, x + 1 < to ? blk + KV4_BLOCK_BYTES : blk};
                    const int most = x + 1 < to ? 32 : 16;
                    ka_blocks<NT>(z, query, two, x + 1 >= plain, [&](int nt, int c) {
                        const int col = nt * 8 + 2 * t + c;
                        return min(most, (col < columns ? seen_by(p0, r0 + col / group) : seen) - first);
                    }, lane);
                }
            }
            __syncwarp();
        }
        /* the stretch's next unit is on its way while this one's result is written and, where it is shared, put together */
        const Segment done = s;
        cur += (unsigned)(s.x1 - s.x0);
        const bool go_on = cur < end;
        if (go_on) {
            s = segment(cur);
#pragma unroll
            for (int i = 0; i < KA_STAGES - 1; i++) fetch(s, i);
        }

        /* the m term of a group to the lanes that hold its channels */
        float m_term[NT][2][4];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
#pragma unroll
                for (int j = 0; j < 4; j++) m_term[nt][c][j] = __shfl_sync(S2P_FULL_MASK, z.om[nt][c], 4 * j + t);
            }
        auto channels = [&](int nt, int c, int j) { /* 32 j + 4 g .. + 3 of column 8 nt + 2 t + c */
            const float m = m_term[nt][c][j];
            return make_float4(fmaf(z.o[nt][2 * j][c], 16777216.0f, m), fmaf(z.o[nt][2 * j][c + 2], 1048576.0f, m), fmaf(z.o[nt][2 * j + 1][c], 16777216.0f, m),
                               fmaf(z.o[nt][2 * j + 1][c + 2], 1048576.0f, m));
        };
        const bool whole = done.x0 == 0 && done.x1 == done.blocks;
        const int w0 = done.w0, w1 = done.w1;
        const size_t slot = 2 * (size_t)worker + (done.x0 == 0 ? 1 : 0);
        unsigned* arrived = parts.arrived + (size_t)row * cache.kv_heads + head;
        auto out_of = [&](int col) { return out + (size_t)(row + col / group) * q_stride + (size_t)(head * group + col % group) * 128; };

        if (by_warp) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const int col = nt * 8 + 2 * t + c;
                    if (col >= columns) continue;
                    if (whole) {
                        __nv_bfloat16* to = out_of(col) + 4 * g;
#pragma unroll
                        for (int j = 0; j < 4; j++) ka_store(to + 32 * j, channels(nt, c, j), z.om[nt][2 + c]);
                    } else {
                        float* to = parts.o + (slot * COLS + col) * 128 + 4 * g;
#pragma unroll
                        for (int j = 0; j < 4; j++) *reinterpret_cast<float4*>(to + 32 * j) = channels(nt, c, j);
                        if (g == 0) {
                            parts.max[slot * COLS + col] = ka_base(z, query, nt, c);
                            parts.sum[slot * COLS + col] = z.om[nt][2 + c];
                        }
                    }
                }
            if (!whole) {
                __syncwarp();
                int last = 0;
                if (lane == 0) last = kv4_arrive(arrived, w1 - w0);
                if (__shfl_sync(S2P_FULL_MASK, last, 0)) {
                    __syncwarp(); /* what lane 0 has acquired, for all: a shuffle does not order memory */
                    for (int base = 0; base < columns; base += KA_PASS) {
                        float top[KA_PASS], sum[KA_PASS];
                        float4 acc[KA_PASS];
                        ka_gather<COLS>(parts, w0, w0, 1, w1, base, columns, lane, top, sum, acc);
#pragma unroll
                        for (int k = 0; k < KA_PASS; k++)
                            if (base + k < columns) ka_store(out_of(base + k) + 4 * lane, acc[k], sum[k]);
                    }
                }
            }
        } else {
            /* Four columns at a time through shared memory.  First the warps' own results; then, in the last CTA of a shared unit, what
             * each warp has gathered of the CTAs' results. */
            const int col = tid >> 6, dim = (tid & 63) * 2; /* threads 0 .. 255 */
            auto together = [&](int base, bool to_out) {
                __syncthreads();
                const int at = base + col;
                if (col < KA_PASS && at < columns) {
                    float top = -INFINITY, sum = 0.0f, a0 = 0.0f, a1 = 0.0f;
#pragma unroll
                    for (int w = 0; w < KA_WARPS; w++) top = fmaxf(top, sh_max[w][at]);
                    const float base2 = top == -INFINITY ? 0.0f : top;
#pragma unroll
                    for (int w = 0; w < KA_WARPS; w++) {
                        const float scale = ka_exp2(sh_max[w][at] - base2);
                        const float2 v = *reinterpret_cast<const float2*>(merge + (w * KA_PASS + col) * 128 + dim);
                        sum = fmaf(sh_sum[w][at], scale, sum);
                        a0 = fmaf(v.x, scale, a0);
                        a1 = fmaf(v.y, scale, a1);
                    }
                    if (to_out) {
                        const float r = sum == 0.0f ? 0.0f : 1.0f / sum;
                        *reinterpret_cast<__nv_bfloat162*>(out_of(at) + dim) = __floats2bfloat162_rn(a0 * r, a1 * r);
                    } else {
                        if ((tid & 63) == 0) {
                            parts.max[slot * COLS + at] = top;
                            parts.sum[slot * COLS + at] = sum;
                        }
                        *reinterpret_cast<float2*>(parts.o + (slot * COLS + at) * 128 + dim) = make_float2(a0, a1);
                    }
                }
                __syncthreads();
            };
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < 2; c++)
                    if (g == 0) {
                        sh_max[warp][nt * 8 + 2 * t + c] = ka_base(z, query, nt, c);
                        sh_sum[warp][nt * 8 + 2 * t + c] = z.om[nt][2 + c];
                    }
#pragma unroll
            for (int pass = 0; pass < 2 * NT; pass++) {
                if (pass * KA_PASS >= columns) break;
                if ((t >> 1) == (pass & 1)) {
#pragma unroll
                    for (int c = 0; c < 2; c++)
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            *reinterpret_cast<float4*>(merge + (warp * KA_PASS + 2 * (t & 1) + c) * 128 + 32 * j + 4 * g) = channels(pass >> 1, c, j);
                }
                together(pass * KA_PASS, whole);
            }
            if (!whole) {
                if (tid == 0) sh_last = kv4_arrive(arrived, w1 - w0);
                __syncthreads();
                if (sh_last) {
                    for (int base = 0; base < columns; base += KA_PASS) {
                        float top[KA_PASS], sum[KA_PASS];
                        float4 acc[KA_PASS];
                        ka_gather<COLS>(parts, w0, w0 + warp, KA_WARPS, w1, base, columns, lane, top, sum, acc);
#pragma unroll
                        for (int k = 0; k < KA_PASS; k++) {
                            if (base + k < COLS && lane == 0) {
                                sh_max[warp][base + k] = top[k];
                                sh_sum[warp][base + k] = sum[k];
                            }
                            *reinterpret_cast<float4*>(merge + (warp * KA_PASS + k) * 128 + 4 * lane) = acc[k];
                        }
                        together(base, true);
                    }
                }
                __syncthreads();
            }
        }
        if (!go_on) break;
    }
}

template <int NT>
static cudaError_t launch_attn(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int layer, int few, const void* q, void* out, cudaStream_t st) {
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
    unsigned char* area = static_cast<unsigned char*>(c->work) + KV4_STATUS_BYTES;
    p.arrived = reinterpret_cast<unsigned*>(area + KV4_AREA_BYTES);
    p.o = reinterpret_cast<float*>(area);
    p.max = p.o + (size_t)KV4_PARTS * 128;
    p.sum = p.max + KV4_PARTS;
    const int group = c->q_heads / c->kv_heads, grid = sms[dev], most = KV4_PARTS / (2 * KA_WARPS * 8 * NT);
    return launch_after(k_kv4_attn<NT>, dim3((unsigned)(grid < most ? grid : most)), KA_THREADS, smem, st, kv4_view(*c, layer), kv4_rows(*b), few,
                        group, 8 * NT > group ? 8 * NT / group : 1, static_cast<const __nv_bfloat16*>(q), static_cast<__nv_bfloat16*>(out), p);
}

extern "C" cudaError_t kv4_attention(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int layer, const void* q, void* out, cudaStream_t st) {
    const int group = c->q_heads / c->kv_heads, most = b->max_rows < b->rows ? b->max_rows : b->rows;
    int few = INT_MAX;
    if (most * group > KA_FEW && kv4_slices_serve(c, b)) {
        few = b->n == 1 ? 0 : KA_FEW_BESIDE / group; /* the rows of an entry are known on the device alone: a batch of several may need both kernels */
        const cudaError_t e = kv4_slices(c, b, layer, few, q, out, st);
        if (e != cudaSuccess || !few) return e;
    }
    /* Next to slices most entries bring a single token, and those of a few rows read their sequence a few times.  A row's query heads of a kv
     * head are not divided. */
    const bool one = group <= 8 && (few < most || most * group <= 8);
    return one ? launch_attn<1>(c, b, layer, few, q, out, st) : launch_attn<2>(c, b, layer, few, q, out, st);
}

}  // namespace s2p
