/* What the kernels of the paged 4-bit cache share: its addressing and its quantiser.  The layout is the one that
 * include/s2p_b200_ext.h documents. */
#pragma once
#include "common.cuh"
#include "kv4.h"
#include "launch.cuh"

namespace s2p {

constexpr int KV4_PARAMS_K = 2048, KV4_PARAMS_V = 2304; /* byte offsets inside a block; s first, m behind it */

/* one layer of a cache, as a kernel sees it */
struct Kv4View {
    unsigned char* pages; /* of page 0, head 0 of the layer */
    size_t page_stride;
    const int32_t* table;
    int n_pages, kv_heads, q_heads, max_seqs, stride;
};
static inline Kv4View kv4_view(const s2p_b200_kv4& c, int layer) {
    Kv4View v;
    const size_t plane = (size_t)c.kv_heads * KV4_HEAD_BYTES;
    v.pages = static_cast<unsigned char*>(c.pages) + (size_t)layer * plane;
    v.page_stride = (size_t)c.layers * plane;
    v.table = c.table;
    v.n_pages = c.n_pages; v.kv_heads = c.kv_heads; v.q_heads = c.q_heads; v.max_seqs = c.max_seqs; v.stride = c.table_stride;
    return v;
}
struct Kv4Rows {
    const int32_t *seqs, *row0, *pos0;
    int n, rows;
};
static inline Kv4Rows kv4_rows(const s2p_b200_kv4_batch& b) { return Kv4Rows{b.seqs, b.row0, b.pos0, b.n, b.rows}; }

/* page of position `pos` of a sequence, or -1; the position may be any number */
__device__ __forceinline__ int kv4_page(const Kv4View& v, int seq, int pos) {
    if ((unsigned)seq >= (unsigned)v.max_seqs || pos < 0 || pos / S2P_B200_KV4_PAGE >= v.stride) return -1;
    const int page = v.table[(size_t)seq * v.stride + pos / S2P_B200_KV4_PAGE];
    return (unsigned)page < (unsigned)v.n_pages ? page : -1;
}
__device__ __forceinline__ unsigned char* kv4_block(const Kv4View& v, int page, int head, int pos) {
    return v.pages + (size_t)page * v.page_stride + (size_t)head * KV4_HEAD_BYTES + (size_t)((pos % S2P_B200_KV4_PAGE) / 16) * KV4_BLOCK_BYTES;
}

/* The sequence and position of row r, position -1 if its entry stores and sees nothing; false if no entry brings it. */
__device__ __forceinline__ bool kv4_find(const Kv4View& v, const Kv4Rows& b, int r, int& seq, int& pos) {
    int lo = 0, hi = b.n; /* the last entry with row0 <= r */
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (b.row0[mid] <= r) lo = mid; else hi = mid;
    }
    const int first = b.row0[lo];
    if (r < first || r >= b.row0[lo + 1]) return false;
    seq = b.seqs[lo];
    const int p0 = b.pos0[lo];
    pos = p0 < 0 || p0 > (1 << 30) || (unsigned)seq >= (unsigned)v.max_seqs ? -1 : p0 + (r - first);
    return true;
}

/* A head vector in half a warp: lane l (0 .. 15) has channels 8 l .. 8 l + 7, four lanes a group.  Byte offsets, inside a block, of what the
 * lane has of position i: the four bytes of a key; the two bytes of the first four channels of a value, those of the others 64 on; */
__device__ __forceinline__ int kv4_key_at(int i, int l) { return 64 * i + 16 * (l & 3) + 4 * (l >> 2); }
__device__ __forceinline__ int kv4_value_at(int i, int l) { return 1024 + 512 * (i >> 3) + 128 * (l & 3) + 16 * ((i >> 1) & 3) + 8 * (i & 1) + 2 * (l >> 2); }
/* ... and of s of group j of position i; m of a key 8 bytes on, of a value 128 */
__device__ __forceinline__ int kv4_key_param_at(int i, int j) { return KV4_PARAMS_K + 16 * i + 2 * j; }
__device__ __forceinline__ int kv4_value_param_at(int i, int j) { return KV4_PARAMS_V + 16 * (i >> 1) + 4 * j + 2 * (i & 1); }

/* The lane's codes (low four bits the first channel) and its group's s and m.  `half`: the lanes of the half warp.  fminf and fmaxf pass over
 * a NaN, and clamping it makes it the least. */
__device__ __forceinline__ uint32_t kv4_quantise(float (&v)[8], unsigned half, __half& s_out, __half& m_out) {
    bool fits = true;
#pragma unroll
    for (int i = 0; i < 8; i++) fits = fits && fabsf(v[i]) <= 65504.0f;
    if (!fits)
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = v[i] != v[i] ? v[i] : fminf(fmaxf(v[i], -65504.0f), 65504.0f);
    float lo = fminf(fminf(fminf(v[0], v[1]), fminf(v[2], v[3])), fminf(fminf(v[4], v[5]), fminf(v[6], v[7])));
    float hi = fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
#pragma unroll
    for (int off = 1; off < 4; off <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(half, lo, off));
        hi = fmaxf(hi, __shfl_xor_sync(half, hi, off));
    }
    if (!(lo <= hi)) lo = hi = 0.0f; /* nothing but NaN */
    s_out = __float2half_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.0f));
    m_out = __float2half_rn(lo);
    const float s = __half2float(s_out), m = __half2float(m_out), r = s > 0.0f ? __frcp_rn(s) : 0.0f;
    /* To the nearest whole number, ties to even, by adding 2^23 + 2^22, which leaves it in the low bits.  A quotient by way of the reciprocal
     * has three roundings.  Without a limit it may be large (m is rounded: with 1000.30 the least and a range of 0.01 it is -300), but where it is kept at 0 or 15 the divided
     * one is too, and up to 15 it is off by less than 1e-5: it rounds to the same code unless it lies that close to the middle between two.  Then it is divided after all. */
    const float big = 12582912.0f;
    uint32_t codes = 0;
    float t[8], off = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        t[i] = fminf(fmaxf(__fmul_rn(__fsub_rn(v[i], m), r), 0.0f), 15.0f);
        off = fmaxf(off, fabsf(__fsub_rn(t[i], __fsub_rn(__fadd_rn(t[i], big), big))));
    }
    if (off > 0.4999f)
#pragma unroll
        for (int i = 0; i < 8; i++) t[i] = fminf(fmaxf(__fdiv_rn(__fsub_rn(v[i], m), s), 0.0f), 15.0f);
#pragma unroll
    for (int i = 0; i < 8; i++) codes |= (__float_as_uint(__fadd_rn(t[i], big)) & 15u) << (4 * i);
    return codes;
}

/* One more worker has left its part of a unit that `others` more share; true for the last of them.  By one thread, behind a barrier of
 * those that wrote; the others read behind a barrier.  The counter is back at zero before anybody can need it again. */
__device__ __forceinline__ bool kv4_arrive(unsigned* counter, int others) {
    unsigned old;
    asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(old) : "l"(counter) : "memory");
    if (old != (unsigned)others) return false;
    *counter = 0;
    return true;
}

}  // namespace s2p
