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
#define KV4_MAX_LINE (1 << 29)   /* rows * kv_heads * table_stride of an attention call: its blocks are counted in 32 bits */

/* The workspace: status word | one area for either the partials of a split attention or the lists of the page operators |
 * arrival counters of the split attention, zero between calls.  Everything is at the same place whatever the cache and the
 * number of rows, so that calls on several caches can use one workspace in turn. */
#define KV4_STATUS_BYTES 256
#define KV4_PARTS (2 * 320 * 8 * 8) /* columns of partials: two for each of 8 columns of 8 warps of up to 320 CTAs; 128 + 2 floats each */
#define KV4_SLICE_CTAS 160          /* CTAs of a slices' launch; two partials of 256 rows each, and a few words */
#define KV4_SLICE_PART_FLOATS (256 * (128 + 2) + 8)
#define KV4_AREA_BYTES ((size_t)2 * KV4_SLICE_CTAS * KV4_SLICE_PART_FLOATS * sizeof(float))
#define KV4_MAX_PAGES (1 << 22) /* the page operators keep 8 bytes a page and a little more in the area: a pair of pages per move, a number per page */

#ifdef __cplusplus
namespace s2p {
extern "C" {
#endif

static inline size_t kv4_work_bytes(int rows, int kv_heads) { return KV4_STATUS_BYTES + KV4_AREA_BYTES + (size_t)rows * (size_t)kv_heads * sizeof(unsigned); }
cudaError_t kv4_append(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int layer, const void* qkv, const void* q_norm, const void* k_norm,
                       float eps, float rope_base, void* q, cudaStream_t st);
cudaError_t kv4_read(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int layer, void* k, void* v, cudaStream_t st);
cudaError_t kv4_attention(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int layer, const void* q, void* out, cudaStream_t st);
/* slices of more than `few` rows, where the batch's chunks fit in shared memory */
int kv4_slices_serve(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b);
cudaError_t kv4_slices(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int layer, int few, const void* q, void* out, cudaStream_t st);
cudaError_t kv4_slices_set_wait_ns(unsigned long long ns); /* test hook: deadline of that kernel's bounded waits */
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
