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

/* Byte offset, inside a block, of the two bytes that hold channels 4 l .. 4 l + 3 (lane l's) of position i */
__device__ __forceinline__ int kv4_key_at(int i, int l) { return 64 * i + 16 * ((l & 7) >> 1) + 4 * (l >> 3) + 2 * (l & 1); }
__device__ __forceinline__ int kv4_value_at(int i, int l) {
    return 1024 + 512 * (i >> 3) + 64 * (l & 7) + 16 * ((i >> 1) & 3) + 8 * (i & 1) + 2 * (l >> 3);
}
/* ... and of s of group j of position i; m of a key 8 bytes on, of a value 128 */
__device__ __forceinline__ int kv4_key_param_at(int i, int j) { return KV4_PARAMS_K + 16 * i + 2 * j; }
__device__ __forceinline__ int kv4_value_param_at(int i, int j) { return KV4_PARAMS_V + 16 * (i >> 1) + 4 * j + 2 * (i & 1); }

/* A head vector in a warp, four channels a lane, eight lanes a group: the lane's codes (low four bits the first channel) and
 * its group's s and m.  fminf and fmaxf pass over a NaN, and its code comes out of the conversion as 0. */
__device__ __forceinline__ uint32_t kv4_quantise(const float x[4], __half& s_out, __half& m_out) {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = x[i] != x[i] ? x[i] : fminf(fmaxf(x[i], -65504.0f), 65504.0f);
    float lo = fminf(fminf(v[0], v[1]), fminf(v[2], v[3])), hi = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
#pragma unroll
    for (int off = 1; off < 8; off <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(S2P_FULL_MASK, lo, off));
        hi = fmaxf(hi, __shfl_xor_sync(S2P_FULL_MASK, hi, off));
    }
    if (!(lo <= hi)) lo = hi = 0.0f; /* nothing but NaN */
    s_out = __float2half_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.0f));
    m_out = __float2half_rn(lo);
    const float s = __half2float(s_out), m = __half2float(m_out);
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int c = s > 0.0f ? __float2int_rn(__fdiv_rn(__fsub_rn(v[i], m), s)) : 0;
        codes |= (uint32_t)max(0, min(15, c)) << (4 * i);
    }
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
