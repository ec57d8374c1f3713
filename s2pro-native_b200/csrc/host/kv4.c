/* Paged 4-bit cache: argument checks of the entry points (include/s2p_b200_ext.h); the kernels are in cuda/kv4_*.cu. */
#include <math.h>
#include <stdio.h>
#include "internal.h"
#include "../cuda/kv4.h"

static int misaligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) != 0; }

static int sizes_served(const s2p_b200_kv4* c) {
    return c && c->n_pages > 0 && c->n_pages <= KV4_MAX_PAGES && c->layers > 0 && c->layers <= 1024 && c->kv_heads > 0 && c->kv_heads <= 1024 && c->q_heads > 0 &&
           c->q_heads % c->kv_heads == 0 && c->q_heads / c->kv_heads <= KV4_MAX_GROUP && c->max_seqs > 0 && c->table_stride > 0 &&
           c->table_stride <= KV4_MAX_STRIDE;
}

size_t s2p_b200_kv4_page_bytes(int layers, int kv_heads) {
    if (layers <= 0 || kv_heads <= 0) return 0;
    return (size_t)layers * (size_t)kv_heads * KV4_HEAD_BYTES;
}

size_t s2p_b200_kv4_work_bytes(const s2p_b200_kv4* c, int rows) {
    return !sizes_served(c) || rows < 0 ? 0 : kv4_work_bytes(rows, c->kv_heads);
}

static s2p_status check_cache(const char* what, const s2p_b200_kv4* c, int rows) {
    if (!sizes_served(c)) {
        fprintf(stderr, "[s2pro] %s: the cache's sizes cannot be served (q_heads a multiple of kv_heads, at most %d times as many; up to %d pages, "
                        "%d table entries a sequence)\n", what, KV4_MAX_GROUP, KV4_MAX_PAGES, KV4_MAX_STRIDE);
        return S2P_ERR_INVALID;
    }
    if (!c->pages || !c->table || !c->lens || !c->refs || !c->work) return S2P_ERR_INVALID;
    if (misaligned(c->pages, 128) || misaligned(c->table, 4) || misaligned(c->lens, 4) || misaligned(c->refs, 4) || misaligned(c->work, 256)) {
        fprintf(stderr, "[s2pro] %s: the pool needs 128-byte alignment, the workspace 256\n", what);
        return S2P_ERR_INVALID;
    }
    if (c->work_bytes < s2p_b200_kv4_work_bytes(c, rows)) {
        fprintf(stderr, "[s2pro] %s: a workspace of %zu bytes, %zu are needed for %d rows\n", what, c->work_bytes, s2p_b200_kv4_work_bytes(c, rows), rows);
        return S2P_ERR_INVALID;
    }
    return S2P_OK;
}

/* work_rows: rows that the workspace has to serve (attention keeps counters for them) */
static s2p_status check_batch(const char* what, const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int work_rows) {
    if (!b || b->n < 0 || b->rows < 0 || b->max_rows < 0) return S2P_ERR_INVALID;
    if (b->n > S2P_B200_KV4_MAX_BATCH) {
        fprintf(stderr, "[s2pro] %s: %d sequences in a batch, at most %d are served\n", what, b->n, S2P_B200_KV4_MAX_BATCH);
        return S2P_ERR_INVALID;
    }
    if (b->n > 0 && (!b->seqs || !b->row0 || !b->pos0 || misaligned(b->seqs, 4) || misaligned(b->row0, 4) || misaligned(b->pos0, 4))) return S2P_ERR_INVALID;
    return check_cache(what, c, work_rows);
}

static s2p_status check_layer(const char* what, const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int work_rows, int layer) {
    S2P_TRY(check_batch(what, c, b, work_rows));
    if (layer < 0 || layer >= c->layers) {
        fprintf(stderr, "[s2pro] %s: layer %d of %d\n", what, layer, c->layers);
        return S2P_ERR_INVALID;
    }
    return S2P_OK;
}

/* host lists of sequences: in range, none twice */
static s2p_status check_list(const char* what, const s2p_b200_kv4* c, const int32_t* seqs, int n) {
    for (int i = 0; i < n; i++) {
        if (seqs[i] < 0 || seqs[i] >= c->max_seqs) {
            fprintf(stderr, "[s2pro] %s: sequence %d of %d\n", what, (int)seqs[i], c->max_seqs);
            return S2P_ERR_INVALID;
        }
        for (int j = 0; j < i; j++)
            if (seqs[j] == seqs[i]) {
                fprintf(stderr, "[s2pro] %s: sequence %d stands in the list twice\n", what, (int)seqs[i]);
                return S2P_ERR_INVALID;
            }
    }
    return S2P_OK;
}
static s2p_status check_list_size(const char* what, int n) {
    if (n < 0 || n > S2P_B200_KV4_MAX_LIST) {
        fprintf(stderr, "[s2pro] %s: %d sequences in one call, at most %d are served\n", what, n, S2P_B200_KV4_MAX_LIST);
        return S2P_ERR_INVALID;
    }
    return S2P_OK;
}

s2p_status s2p_b200_kv4_status(const s2p_b200_kv4* c, cudaStream_t stream) {
    S2P_TRY(check_cache("kv4_status", c, 0));
    int code = 0;
    S2P_CUDA_TRY(cudaMemcpyAsync(&code, c->work, sizeof(code), cudaMemcpyDeviceToHost, stream));
    S2P_CUDA_TRY(cudaStreamSynchronize(stream));
    if (!code) return S2P_OK;
    S2P_CUDA_TRY(cudaMemsetAsync(c->work, 0, sizeof(code), stream));
    fprintf(stderr, "[s2pro] kv4_status: a bounded wait of an earlier call gave up (code %d); its rows are lost\n", code);
    return S2P_ERR_INTERNAL;
}

s2p_status s2p_b200_kv4_reserve(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int32_t* info, cudaStream_t stream) {
    S2P_TRY(check_batch("kv4_reserve", c, b, 0));
    if (misaligned(info, 4)) return S2P_ERR_INVALID;
    if (!b->n && !info) return S2P_OK;
    S2P_CUDA_TRY(kv4_reserve(c, b, info, stream));
    return S2P_OK;
}

s2p_status s2p_b200_kv4_append(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int layer, const s2p_bf16* qkv, const s2p_bf16* q_norm,
                               const s2p_bf16* k_norm, float eps, float rope_base, s2p_bf16* q, cudaStream_t stream) {
    S2P_TRY(check_layer("kv4_append", c, b, 0, layer));
    if (!b->n || !b->rows) return S2P_OK;
    if (!qkv || !q || misaligned(qkv, 16) || misaligned(q, 16) || misaligned(q_norm, 8) || misaligned(k_norm, 8)) return S2P_ERR_INVALID;
    if (!(rope_base > 0.0f && rope_base < INFINITY) || !(eps >= 0.0f)) return S2P_ERR_INVALID;
    S2P_CUDA_TRY(kv4_append(c, b, layer, qkv, q_norm, k_norm, eps, rope_base, q, stream));
    return S2P_OK;
}

s2p_status s2p_b200_kv4_attention(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int layer, const s2p_bf16* q, s2p_bf16* out,
                                  cudaStream_t stream) {
    S2P_TRY(check_layer("kv4_attention", c, b, b && b->rows > 0 ? b->rows : 0, layer));
    if (!b->n || !b->rows) return S2P_OK;
    if (!q || !out || misaligned(q, 16) || misaligned(out, 16)) return S2P_ERR_INVALID;
    if ((double)b->rows * c->kv_heads * c->table_stride > (double)KV4_MAX_LINE) {
        fprintf(stderr, "[s2pro] kv4_attention: rows * kv_heads * table_stride is above %d: split the batch\n", KV4_MAX_LINE);
        return S2P_ERR_INVALID;
    }
    S2P_CUDA_TRY(kv4_attention(c, b, layer, q, out, stream));
    return S2P_OK;
}

s2p_status s2p_b200_kv4_read(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int layer, s2p_bf16* k, s2p_bf16* v, cudaStream_t stream) {
    S2P_TRY(check_layer("kv4_read", c, b, 0, layer));
    if (!b->n || !b->rows) return S2P_OK;
    if (!k || !v || misaligned(k, 16) || misaligned(v, 16)) return S2P_ERR_INVALID;
    S2P_CUDA_TRY(kv4_read(c, b, layer, k, v, stream));
    return S2P_OK;
}

s2p_status s2p_b200_kv4_fork(const s2p_b200_kv4* c, const int32_t* parents, const int32_t* children, const int32_t* tokens, int n, int32_t* info,
                             cudaStream_t stream) {
    S2P_TRY(check_cache("kv4_fork", c, 0));
    S2P_TRY(check_list_size("kv4_fork", n));
    if (misaligned(info, 4)) return S2P_ERR_INVALID;
    if (!n && !info) return S2P_OK;
    if (n && (!parents || !children || !tokens)) return S2P_ERR_INVALID;
    S2P_TRY(check_list("kv4_fork", c, children, n));
    for (int i = 0; i < n; i++) {
        if (parents[i] < 0 || parents[i] >= c->max_seqs || tokens[i] < -1) return S2P_ERR_INVALID;
        for (int j = 0; j < n; j++)
            if (parents[i] == children[j]) {
                fprintf(stderr, "[s2pro] kv4_fork: sequence %d is a parent and a child\n", (int)parents[i]);
                return S2P_ERR_INVALID;
            }
    }
    S2P_CUDA_TRY(kv4_fork(c, parents, children, tokens, n, info, stream));
    return S2P_OK;
}

s2p_status s2p_b200_kv4_release(const s2p_b200_kv4* c, const int32_t* seqs, int n, cudaStream_t stream) {
    S2P_TRY(check_cache("kv4_release", c, 0));
    S2P_TRY(check_list_size("kv4_release", n));
    if (!n) return S2P_OK;
    if (!seqs) return S2P_ERR_INVALID;
    S2P_TRY(check_list("kv4_release", c, seqs, n));
    S2P_CUDA_TRY(kv4_release(c, seqs, n, stream));
    return S2P_OK;
}

s2p_status s2p_b200_kv4_compact(const s2p_b200_kv4* c, int32_t* info, cudaStream_t stream) {
    S2P_TRY(check_cache("kv4_compact", c, 0));
    if (misaligned(info, 4)) return S2P_ERR_INVALID;
    S2P_CUDA_TRY(kv4_compact(c, info, stream));
    return S2P_OK;
}
