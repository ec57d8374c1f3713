/* Launchers of the paged 4-bit cache (include/s2p_b200_ext.h), called by host/kv4.c, which checks the arguments.
 * None of this is exported. */
#ifndef S2P_KV4_H
#define S2P_KV4_H

#include "s2p_b200_ext.h"

/* bytes of a block of 16 positions, and of the four of a page, of one kv head */
#define KV4_BLOCK_BYTES 2560
#define KV4_HEAD_BYTES (4 * KV4_BLOCK_BYTES)
#define KV4_MAX_GROUP 16         /* query heads of a kv head */
#define KV4_MAX_STRIDE (1 << 24) /* table entries of a sequence: positions stay below 2^30 */

/* The workspace: status word | arrival counters of the split attention, zero between calls | one area for either the partials
 * of a split attention or the lists of the page operators. */
#define KV4_MAX_CTAS 320         /* CTAs that may leave partials, two each */
#define KV4_PART_COLS 16         /* (row, head) columns of a partial */
#define KV4_PART_FLOATS (KV4_PART_COLS * (128 + 2))
#define KV4_STATUS_BYTES 256

#ifdef __cplusplus
namespace s2p {
extern "C" {
#endif

size_t kv4_counter_bytes(int rows, int kv_heads);
cudaError_t kv4_append(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int layer, const void* qkv, const void* q_norm, const void* k_norm,
                       float eps, float rope_base, void* q, cudaStream_t st);
cudaError_t kv4_read(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int layer, void* k, void* v, cudaStream_t st);
cudaError_t kv4_attention(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int layer, const void* q, void* out, cudaStream_t st);
cudaError_t kv4_reserve(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int32_t* info, cudaStream_t st);
cudaError_t kv4_fork(const s2p_b200_kv4* c, const int32_t* parents, const int32_t* children, const int32_t* tokens, int n, int32_t* info,
                     cudaStream_t st);
cudaError_t kv4_release(const s2p_b200_kv4* c, const int32_t* seqs, int n, cudaStream_t st);
cudaError_t kv4_compact(const s2p_b200_kv4* c, int32_t* info, cudaStream_t st);

#ifdef __cplusplus
} /* extern "C" */
} /* namespace s2p */
#endif
#endif
