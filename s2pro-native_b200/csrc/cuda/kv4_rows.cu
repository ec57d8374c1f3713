/* Paged 4-bit cache: rows in and out.
 *
 * append: per head vector x of a row at position p, y = x * rsqrt(mean(x^2) + eps) * w; channel pairs (2 i, 2 i + 1) turned by the
 * angle p * base^(-2 i / 128); queries rounded to bf16, keys (turned) and values (as they come) quantised in groups of 32.
 * Half a warp holds a head vector, eight channels a lane: the norm is one shuffle tree, the pairs are inside a lane, a group is four
 * lanes.  All of it is in 32 bits up to the one rounding of the result; the angle is reduced in 64 (at position 32768 the fastest pair has
 * turned 5215 times: 32 bits would leave it 2e-3 off).
 *
 * Few rows are bound by latency (32 query and 8 kv heads, append and read of 1 to 32 rows: 7.2 us, launches included), many by the issue of instructions: append of 2055 rows,
 * 44.7 MB, 18.9 us, of which HBM would take 6.9; 60% of the issue slots are busy.  (With a warp to a vector, 193 instructions each, append and read 41 us; now 25.8.)  Read of 2055
 * rows, 11 MB, 8.9 us.  The row grid below was measured on the two together. */
#include <math.h>
#include "kv4.cuh"

namespace s2p {

constexpr int KV4_ROW_WARPS = 8, KV4_ROWS = 4, KV4_AHEAD = 3; /* warps and rows of a CTA; pairs of vectors whose loads a warp has under way */

/* cosine and sine of a pair at position pos; per_position: the turns that it makes from one to the next */
__device__ __forceinline__ float2 kv4_turn(int pos, double per_position) {
    double turns = (double)pos * per_position;
    turns -= rint(turns);
    float s, c;
    sincospif(2.0f * (float)turns, &s, &c);
    return make_float2(c, s);
}

struct Kv4Place { int found, pos, page; }; /* of a row: whether an entry brings it, its position or -1, the page or -1 */
__device__ __forceinline__ Kv4Place kv4_place(const Kv4View& cache, const Kv4Rows& b, int row) {
    Kv4Place p;
    int seq = -1;
    p.pos = -1;
    p.found = row < b.rows && kv4_find(cache, b, row, seq, p.pos);
    p.page = p.found && p.pos >= 0 ? kv4_page(cache, seq, p.pos) : -1;
    return p;
}

/* A CTA has `rows` (up to KV4_ROWS) consecutive rows, whose places and angles it works out once, and its warps their pairs of head vectors in turn. */
__global__ void __launch_bounds__(KV4_ROW_WARPS * 32, 4)
k_kv4_append(Kv4View cache, Kv4Rows b, int rows, const __nv_bfloat16* qkv, const __nv_bfloat16* q_norm, const __nv_bfloat16* k_norm, float eps,
             double per_pair /* log2(base) / 64 */, __nv_bfloat16* q) {
    __shared__ __align__(16) float2 turn[KV4_ROWS][64];
    __shared__ Kv4Place place[KV4_ROWS];
    const int row0 = blockIdx.x * rows, l = threadIdx.x & 15, second = (threadIdx.x >> 4) & 1;
    const unsigned half = 0xFFFFu << (16 * second);
    const int heads = cache.q_heads + 2 * cache.kv_heads, step = KV4_ROW_WARPS * gridDim.y, first = blockIdx.y * KV4_ROW_WARPS + (threadIdx.x >> 5);
    static_assert(KV4_ROW_WARPS * 32 % 64 == 0, "a thread's angles are of one pair of channels");
    const double per_position = exp2(-(double)(threadIdx.x & 63) * per_pair) * 0.15915494309189533577; /* 1 / 2 pi */
    grid_wait();
    grid_release();
    if (threadIdx.x < rows) place[threadIdx.x] = kv4_place(cache, b, row0 + threadIdx.x);
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * rows; i += KV4_ROW_WARPS * 32) turn[i >> 6][i & 63] = kv4_turn(max(place[i >> 6].pos, 0), per_position);
    __syncthreads();
    for (int r = 0; r < rows; r++) {
        const int pos = place[r].pos, page = place[r].page;
        if (!place[r].found) continue;
        const uint4* from = reinterpret_cast<const uint4*>(qkv + (size_t)(row0 + r) * heads * 128) + l;
        for (int i0 = first; 2 * i0 < heads; i0 += KV4_AHEAD * step) {
            uint4 raws[KV4_AHEAD];
#pragma unroll
            for (int k = 0; k < KV4_AHEAD; k++) {
                const int head = 2 * (i0 + k * step) + second;
                raws[k] = head < heads && pos >= 0 ? from[head * 16] : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int k = 0; k < KV4_AHEAD; k++) {
                const int head = 2 * (i0 + k * step) + second;
                const bool is_q = head < cache.q_heads, is_v = head >= cache.q_heads + cache.kv_heads;
                if (head >= heads || (!is_q && page < 0)) continue;
                const uint4 raw = raws[k];
                float x[8] = {bf_lo(raw.x), bf_hi(raw.x), bf_lo(raw.y), bf_hi(raw.y), bf_lo(raw.z), bf_hi(raw.z), bf_lo(raw.w), bf_hi(raw.w)};
                if (!is_v) {
                    const __nv_bfloat16* w = is_q ? q_norm : k_norm;
                    if (w) {
                        float sum = 0.0f;
#pragma unroll
                        for (int i = 0; i < 8; i++) sum = fmaf(x[i], x[i], sum);
#pragma unroll
                        for (int off = 1; off < 16; off <<= 1) sum += __shfl_xor_sync(half, sum, off);
                        const float n = rsqrtf(sum * (1.0f / 128.0f) + eps);
                        const uint2 g0 = reinterpret_cast<const uint2*>(w)[2 * l], g1 = reinterpret_cast<const uint2*>(w)[2 * l + 1];
                        const float g[8] = {bf_lo(g0.x), bf_hi(g0.x), bf_lo(g0.y), bf_hi(g0.y), bf_lo(g1.x), bf_hi(g1.x), bf_lo(g1.y), bf_hi(g1.y)};
#pragma unroll
                        for (int i = 0; i < 8; i++) x[i] *= n * g[i];
                    }
                    const float4 t0 = reinterpret_cast<const float4*>(turn[r])[2 * l], t1 = reinterpret_cast<const float4*>(turn[r])[2 * l + 1];
                    const float c[4] = {t0.x, t0.z, t1.x, t1.z}, s[4] = {t0.y, t0.w, t1.y, t1.w};
#pragma unroll
                    for (int h = 0; h < 4; h++) {
                        const float a = x[2 * h], d = x[2 * h + 1];
                        x[2 * h] = a * c[h] - d * s[h];
                        x[2 * h + 1] = d * c[h] + a * s[h];
                    }
                }
                if (is_q) {
                    uint32_t y[4];
#pragma unroll
                    for (int h = 0; h < 4; h++) {
                        const __nv_bfloat162 z = __floats2bfloat162_rn(x[2 * h], x[2 * h + 1]);
                        y[h] = *reinterpret_cast<const uint32_t*>(&z);
                    }
                    reinterpret_cast<uint4*>(q + ((size_t)(row0 + r) * cache.q_heads + head) * 128)[l] = make_uint4(y[0], y[1], y[2], y[3]);
                    continue;
                }
                __half s, m;
                const uint32_t codes = kv4_quantise(x, half, s, m);
                const int in = pos % 16, j = l >> 2;
                unsigned char* block = kv4_block(cache, page, head - cache.q_heads - (is_v ? cache.kv_heads : 0), pos);
                if (is_v) {
                    unsigned char* at = block + kv4_value_at(in, l);
                    *reinterpret_cast<uint16_t*>(at) = (uint16_t)codes;
                    *reinterpret_cast<uint16_t*>(at + 64) = (uint16_t)(codes >> 16);
                } else *reinterpret_cast<uint32_t*>(block + kv4_key_at(in, l)) = codes;
                if ((l & 3) == 0) {
                    unsigned char* at = block + (is_v ? kv4_value_param_at(in, j) : kv4_key_param_at(in, j));
                    *reinterpret_cast<__half*>(at) = s;
                    *reinterpret_cast<__half*>(at + (is_v ? 128 : 8)) = m;
                }
            }
        }
    }
}

/* Rows to a CTA and CTAs to them: as many rows as leave the CTAs one wave of four to an SM, up to four (2055 rows: 1, 2, 4, 8 to a CTA 31, 27.9, 26, 39 us;
 * 1000 rows: 2 to a CTA 15, 4 in two CTAs 19.4), several CTAs where there are few. */
struct Kv4RowGrid { dim3 grid; int rows; };
static Kv4RowGrid kv4_row_grid(int rows, int vectors) {
    Kv4RowGrid g;
    g.rows = rows <= 3 * 592 ? (rows + 591) / 592 : KV4_ROWS;
    const int x = (rows + g.rows - 1) / g.rows, most = ((vectors + 1) / 2 + KV4_ROW_WARPS - 1) / KV4_ROW_WARPS;
    const int want = (2 * 148 + x - 1) / x;
    g.grid = dim3((unsigned)x, (unsigned)(want < most ? want : most));
    return g;
}

extern "C" cudaError_t kv4_append(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int layer, const void* qkv, const void* q_norm,
                                  const void* k_norm, float eps, float rope_base, void* q, cudaStream_t st) {
    const Kv4RowGrid g = kv4_row_grid(b->rows, c->q_heads + 2 * c->kv_heads);
    return launch_after(k_kv4_append, g.grid, KV4_ROW_WARPS * 32, 0, st, kv4_view(*c, layer), kv4_rows(*b), g.rows, static_cast<const __nv_bfloat16*>(qkv),
                        static_cast<const __nv_bfloat16*>(q_norm), static_cast<const __nv_bfloat16*>(k_norm), eps > 1e-37f ? eps : 1e-37f /* a row of zeros stays one */, log2((double)rope_base) / 64.0,
                        static_cast<__nv_bfloat16*>(q));
}

/* The inverse of append's stores, its rows and head vectors cut the same way; a pair is a kv head's key and value. */
__global__ void __launch_bounds__(KV4_ROW_WARPS * 32) k_kv4_read(Kv4View cache, Kv4Rows b, int rows, __nv_bfloat16* k_out, __nv_bfloat16* v_out) {
    __shared__ Kv4Place place[KV4_ROWS];
    const int row0 = blockIdx.x * rows, l = threadIdx.x & 15, is_v = (threadIdx.x >> 4) & 1;
    const int step = KV4_ROW_WARPS * gridDim.y, first = blockIdx.y * KV4_ROW_WARPS + (threadIdx.x >> 5);
    grid_wait();
    grid_release();
    if (threadIdx.x < rows) place[threadIdx.x] = kv4_place(cache, b, row0 + threadIdx.x);
    __syncthreads();
    constexpr int AHEAD = 4; /* heads whose loads a warp has under way */
    for (int i0 = first; i0 < rows * cache.kv_heads; i0 += AHEAD * step) {
        uint32_t codes[AHEAD];
        __half s[AHEAD], m[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; k++) {
            const int i = i0 + k * step, r = min(i / cache.kv_heads, rows - 1), head = i - r * cache.kv_heads, pos = place[r].pos, page = place[r].page;
            codes[k] = 0;
            s[k] = m[k] = __half(0.0f);
            if (i < rows * cache.kv_heads && page >= 0) {
                const int in = pos % 16, j = l >> 2;
                const unsigned char* block = kv4_block(cache, page, head, pos);
                const unsigned char* at = block + (is_v ? kv4_value_param_at(in, j) : kv4_key_param_at(in, j));
                s[k] = *reinterpret_cast<const __half*>(at);
                m[k] = *reinterpret_cast<const __half*>(at + (is_v ? 128 : 8));
                if (is_v) codes[k] = *reinterpret_cast<const uint16_t*>(block + kv4_value_at(in, l)) | (uint32_t)*reinterpret_cast<const uint16_t*>(block + kv4_value_at(in, l) + 64) << 16;
                else codes[k] = *reinterpret_cast<const uint32_t*>(block + kv4_key_at(in, l));
            }
        }
#pragma unroll
        for (int k = 0; k < AHEAD; k++) {
            const int i = i0 + k * step, r = min(i / cache.kv_heads, rows - 1), head = i - r * cache.kv_heads;
            if (i >= rows * cache.kv_heads || !place[r].found) continue;
            const float sf = __half2float(s[k]), mf = __half2float(m[k]);
            uint32_t y[4];
#pragma unroll
            for (int h = 0; h < 4; h++) {
                const __nv_bfloat162 z = __floats2bfloat162_rn(fmaf(sf, (float)((codes[k] >> (8 * h)) & 15u), mf), fmaf(sf, (float)((codes[k] >> (8 * h + 4)) & 15u), mf));
                y[h] = *reinterpret_cast<const uint32_t*>(&z);
            }
            reinterpret_cast<uint4*>((is_v ? v_out : k_out) + ((size_t)(row0 + r) * cache.kv_heads + head) * 128)[l] = make_uint4(y[0], y[1], y[2], y[3]);
        }
    }
}

extern "C" cudaError_t kv4_read(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int layer, void* k, void* v, cudaStream_t st) {
    const Kv4RowGrid g = kv4_row_grid(b->rows, 2 * c->kv_heads);
    return launch_after(k_kv4_read, g.grid, KV4_ROW_WARPS * 32, 0, st, kv4_view(*c, layer), kv4_rows(*b), g.rows, static_cast<__nv_bfloat16*>(k),
                        static_cast<__nv_bfloat16*>(v));
}

}  // namespace s2p
