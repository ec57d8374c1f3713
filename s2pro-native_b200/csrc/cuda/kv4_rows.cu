/* Paged 4-bit cache: rows in and out.
 *
 * append: per head vector x of a row at position p, y = x * rsqrt(mean(x^2) + eps) * w; channel pairs (2 i, 2 i + 1) turned by the
 * angle p * base^(-2 i / 128); queries rounded to bf16, keys (turned) and values (as they come) quantised in groups of 32.
 * A warp holds a head vector, four channels a lane: the norm is one shuffle tree, the pairs are inside a lane, a group is eight
 * lanes.  All of it is in 32 bits up to the one rounding of the result; the angle is reduced in 64 (at position 32768 the
 * fastest pair has turned 5215 times: 32 bits would leave it 2e-3 off). */
#include <math.h>
#include "kv4.cuh"

namespace s2p {

constexpr int KV4_ROW_WARPS = 8;

/* cosine and sine of pair i at position pos; per_pair = log2(base) / 64 */
__device__ __forceinline__ float2 kv4_turn(int pos, int i, double per_pair) {
    double turns = (double)pos * exp2(-(double)i * per_pair) * 0.15915494309189533577; /* angle / 2 pi */
    turns -= rint(turns);
    float s, c;
    sincospif(2.0f * (float)turns, &s, &c);
    return make_float2(c, s);
}

__global__ void __launch_bounds__(KV4_ROW_WARPS * 32)
k_kv4_append(Kv4View cache, Kv4Rows b, const __nv_bfloat16* qkv, const __nv_bfloat16* q_norm, const __nv_bfloat16* k_norm, float eps,
             double per_pair, __nv_bfloat16* q) {
    __shared__ float2 turn[64];
    __shared__ int sh[3];
    const int row = blockIdx.x, lane = threadIdx.x & 31;
    const int heads = cache.q_heads + 2 * cache.kv_heads, head = blockIdx.y * KV4_ROW_WARPS + (threadIdx.x >> 5);
    grid_wait();
    grid_release();
    if (threadIdx.x == 0) {
        int seq = -1, pos = -1;
        sh[0] = kv4_find(cache, b, row, seq, pos);
        sh[1] = pos;
        sh[2] = pos >= 0 ? kv4_page(cache, seq, pos) : -1;
    }
    __syncthreads();
    if (!sh[0]) return;
    const int pos = sh[1], page = sh[2];
    if (threadIdx.x < 64) turn[threadIdx.x] = kv4_turn(max(pos, 0), threadIdx.x, per_pair);
    __syncthreads();
    if (head >= heads) return;

    const bool is_q = head < cache.q_heads, is_v = head >= cache.q_heads + cache.kv_heads;
    if (pos < 0) {
        if (is_q) reinterpret_cast<uint2*>(q + ((size_t)row * cache.q_heads + head) * 128)[lane] = make_uint2(0, 0);
        return;
    }
    if (!is_q && page < 0) return;
    const uint2 raw = reinterpret_cast<const uint2*>(qkv + ((size_t)row * heads + head) * 128)[lane];
    float x[4] = {bf_lo(raw.x), bf_hi(raw.x), bf_lo(raw.y), bf_hi(raw.y)};
    if (!is_v) {
        const __nv_bfloat16* w = is_q ? q_norm : k_norm;
        if (w) {
            const float sum = warp_tree_sum(fmaf(x[0], x[0], fmaf(x[1], x[1], fmaf(x[2], x[2], x[3] * x[3]))));
            const float r = 1.0f / sqrtf(sum * (1.0f / 128.0f) + eps);
            const uint2 g = reinterpret_cast<const uint2*>(w)[lane];
            x[0] = x[0] * r * bf_lo(g.x); x[1] = x[1] * r * bf_hi(g.x);
            x[2] = x[2] * r * bf_lo(g.y); x[3] = x[3] * r * bf_hi(g.y);
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float2 t = turn[2 * lane + i];
            const float a = x[2 * i], c = x[2 * i + 1];
            x[2 * i] = a * t.x - c * t.y;
            x[2 * i + 1] = c * t.x + a * t.y;
        }
    }
    if (is_q) {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(x[0], x[1]), hi = __floats2bfloat162_rn(x[2], x[3]);
        reinterpret_cast<uint2*>(q + ((size_t)row * cache.q_heads + head) * 128)[lane] =
            make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
        return;
    }
    __half s, m;
    const uint32_t codes = kv4_quantise(x, s, m);
    const int i = pos % 16, j = lane >> 3;
    unsigned char* block = kv4_block(cache, page, head - cache.q_heads - (is_v ? cache.kv_heads : 0), pos);
    *reinterpret_cast<uint16_t*>(block + (is_v ? kv4_value_at(i, lane) : kv4_key_at(i, lane))) = (uint16_t)codes;
    if ((lane & 7) == 0) {
        unsigned char* at = block + (is_v ? kv4_value_param_at(i, j) : kv4_key_param_at(i, j));
        *reinterpret_cast<__half*>(at) = s;
        *reinterpret_cast<__half*>(at + (is_v ? 128 : 8)) = m;
    }
}

extern "C" cudaError_t kv4_append(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int layer, const void* qkv, const void* q_norm,
                                  const void* k_norm, float eps, float rope_base, void* q, cudaStream_t st) {
    const int heads = c->q_heads + 2 * c->kv_heads;
    return launch_after(k_kv4_append, dim3((unsigned)b->rows, (unsigned)((heads + KV4_ROW_WARPS - 1) / KV4_ROW_WARPS)), KV4_ROW_WARPS * 32, 0, st,
                        kv4_view(*c, layer), kv4_rows(*b), static_cast<const __nv_bfloat16*>(qkv), static_cast<const __nv_bfloat16*>(q_norm),
                        static_cast<const __nv_bfloat16*>(k_norm), eps, log2((double)rope_base) / 64.0, static_cast<__nv_bfloat16*>(q));
}

/* One warp per (row, kv head, keys or values): the inverse of append's stores. */
__global__ void __launch_bounds__(KV4_ROW_WARPS * 32) k_kv4_read(Kv4View cache, Kv4Rows b, __nv_bfloat16* k, __nv_bfloat16* v) {
    const int row = blockIdx.x, lane = threadIdx.x & 31, unit = blockIdx.y * KV4_ROW_WARPS + (threadIdx.x >> 5);
    if (unit >= 2 * cache.kv_heads) return;
    grid_wait();
    grid_release();
    int seq = -1, pos = -1;
    if (!kv4_find(cache, b, row, seq, pos)) return;
    const int head = unit >> 1, is_v = unit & 1, page = pos >= 0 ? kv4_page(cache, seq, pos) : -1;
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (page >= 0) {
        const int i = pos % 16, j = lane >> 3;
        const unsigned char* block = kv4_block(cache, page, head, pos);
        const uint32_t codes = *reinterpret_cast<const uint16_t*>(block + (is_v ? kv4_value_at(i, lane) : kv4_key_at(i, lane)));
        const unsigned char* at = block + (is_v ? kv4_value_param_at(i, j) : kv4_key_param_at(i, j));
        const float s = __half2float(*reinterpret_cast<const __half*>(at)), m = __half2float(*reinterpret_cast<const __half*>(at + (is_v ? 128 : 8)));
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = fmaf(s, (float)((codes >> (4 * e)) & 15u), m);
    }
    const __nv_bfloat162 lo = __floats2bfloat162_rn(x[0], x[1]), hi = __floats2bfloat162_rn(x[2], x[3]);
    reinterpret_cast<uint2*>((is_v ? v : k) + ((size_t)row * cache.kv_heads + head) * 128)[lane] =
        make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}

extern "C" cudaError_t kv4_read(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int layer, void* k, void* v, cudaStream_t st) {
    return launch_after(k_kv4_read, dim3((unsigned)b->rows, (unsigned)((2 * c->kv_heads + KV4_ROW_WARPS - 1) / KV4_ROW_WARPS)), KV4_ROW_WARPS * 32, 0,
                        st, kv4_view(*c, layer), kv4_rows(*b), static_cast<__nv_bfloat16*>(k), static_cast<__nv_bfloat16*>(v));
}

}  // namespace s2p
