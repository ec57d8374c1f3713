/* s2pro-b200 — additive entry points that have no counterpart in the
 * reference's headers.  Everything the reference's callers use is in
 * s2p_b200_abi.h; a drop-in build never needs this file. */
#ifndef S2P_B200_EXT_H
#define S2P_B200_EXT_H

#include "s2p_b200_abi.h"

#ifdef __cplusplus
extern "C" {
#endif
/* the library is built with hidden visibility; only what is declared here is exported */
#pragma GCC visibility push(default)

/* Library identification: "s2pro-b200 <version> sm_100a". */
const char* s2p_b200_version(void);

/* Measurement hooks (no counterpart in the reference). */
typedef struct {
    uint64_t frames_decoded;        /* session-frames produced since load */
    int n_slow_layers;              /* backbone depth found in the checkpoint */
    int last_tick_rows;             /* rows of the most recent tick */
    int last_tick_fused;            /* 1 = batch-1 fused stages, 0 = general sequence */
    int last_tick_graph;            /* 1 = replayed from a captured CUDA graph */
    int last_tick_kernels;          /* kernel launches of the most recent tick */
    float last_tick_device_ms;      /* device time of the most recent tick (events on the model stream) */
    size_t upload_bytes;            /* host->device bytes per tick */
    size_t download_bytes;          /* device->host bytes per tick */
    double weight_bytes_per_frame;  /* quantised weight + scale bytes one batch-1 frame streams */
    double kv_bytes_per_token;      /* KV bytes one session reads per cached token per frame */
    int last_tick_persistent;       /* 1 = the whole tick ran as one persistent cooperative kernel */
} s2p_b200_stats;

s2p_status s2p_b200_model_stats(const s2p_model* m, s2p_b200_stats* out);

/* Stage trace of the persistent tick kernel (no counterpart in the reference).  With
 * S2P_TICK_TRACE=1 in the environment at model load, CTA 0 of every persistent tick
 * records sixteen 64-bit words per stage; this call copies those of the most recent tick:
 * out[16 * stage + w].  Words 0..3 are SM-clock stamps: stage entered, activation staged
 * (GEMV stages; 0 otherwise), own work done, grid barrier passed (or stage left where
 * the stage ends without one).  Words 4..7 are SM-clock sums of thread 0's streaming
 * role (waiting for weight chunks, multiplying) and of fold warp 0 (waiting for
 * partial sums, folding); words 8..15 are the SM clock at which each of the eight
 * streaming warps was through.  types[stage] = stage kind (0 frame start, 1 GEMV,
 * 2 backbone attention, 3 fast-AR attention, 4 sampler, 5 frame end).  *n_stages
 * receives the stage count; at most max_stages stages are written.  S2P_ERR_STATE if
 * tracing is off or no persistent tick has run. */
s2p_status s2p_b200_model_tick_trace(s2p_model* m, uint64_t* out, int32_t* types, int max_stages, int* n_stages);
/* Per-CTA stamps of the same tick, in nanoseconds of the GPU's global timer:
 * fold_done_ns[stage * n_ctas + cta] = the CTA's last output of the stage was published
 * (for stages without a GEMV: the stage body returned), staged_ns[...] = its
 * activation vector of a GEMV stage was staged in shared memory (0 elsewhere).  The
 * difference between the latest fold_done of stage s and a CTA's staged stamp of stage
 * s+1 is the hand-off latency between two GEMV stages.  Both arrays must hold
 * n_stages * n_ctas words (S2P_ERR_INVALID with the two counts filled in otherwise). */
s2p_status s2p_b200_model_tick_trace_ctas(s2p_model* m, uint64_t* fold_done_ns, uint64_t* staged_ns, int max_stages, int max_ctas,
                                          int* n_stages, int* n_ctas);
/* The stream every tick of this model is issued on (for external event timing). */
cudaStream_t s2p_b200_model_stream(s2p_model* m);

/* Tensor-parallel batch-1 decode over 2, 4 or 8 GPUs of one node (no counterpart in the
 * reference, which runs one GPU per process and has no sharded path).  One process per GPU
 * loads the same checkpoint, exports a handle to its exchange arena, receives the handles of
 * all ranks (any transport: the caller exchanges 64-byte blobs), and attaches before creating
 * sessions.  From then on every rank must issue the same API calls with the same arguments in
 * the same order; the persistent tick kernels of the ranks split the rows of every matrix
 * between them, store each stage's outputs into every rank's arena over NVLink and meet at a
 * barrier that spans the ranks.  Every row is still computed by one thread block with the
 * single-GPU arithmetic, so the frames are bit-identical to a single-GPU run.  Each kv head's
 * cache is kept current only on the rank that attends over it.  Consequences, enforced with
 * S2P_ERR_UNSUPPORTED and a message rather than left to produce wrong frames:
 *  - s2p_session_kv_save is refused for a tensor-parallel session (the blob would be incomplete);
 *  - a tick with decoding rows that cannot run as the persistent kernel is refused: more than one
 *    session, or any tick after the persistent kernel was disabled because one of its bounded waits
 *    gave up (that tick returned S2P_ERR_INTERNAL).  The single-GPU fallbacks of an unsharded model
 *    do not exist here.
 * Prefill is replicated on every rank. */
#define S2P_B200_TP_HANDLE_BYTES 64
s2p_status s2p_b200_model_tp_export(s2p_model* m, void* handle_out);
s2p_status s2p_b200_model_tp_attach(s2p_model* m, int rank, int world, const void* handles);

/* Decode attention that never asks the driver for memory.  (No counterpart in the
 * reference: its split-K attention takes a caller-allocated scratch pointer.)
 *
 * Some hosts of this library may not allocate device memory while they run: a
 * real-time audio worker whose tick must never wait on cudaMalloc / cudaFree (both
 * serialise against every stream of the device, the vocoder's included), or an
 * embedding application that gives a plug-in no memory pool of its own.  For them
 * this entry point computes the split-K GQA decode attention of ONE query row —
 * 32 query heads over 8 kv heads of width 128, bf16 cache planes
 * [kv_heads, max_seq, 128], attending positions 0..pos — with its scratch (split
 * partials and arrival counters) in a fixed ~2.1 MB array built into the library.
 * The result equals the library's regular split-K decode attention bit for bit.
 *
 * Limits and rules:
 *  - pos + 1 <= 8192 cached positions; anything larger is refused with S2P_ERR_INVALID
 *    and a message (use the regular path, whose scratch is sized at model load);
 *  - the first call on each device looks up the array's device address
 *    (cudaGetSymbolAddress); make that first call before starting any stream capture;
 *  - all calls share the one array: calls that can overlap on the GPU (different
 *    streams, or two host threads) race — issue them on one stream;
 *  - no cudaMalloc, cudaFree or allocating library routine is called, ever. */
s2p_status s2p_b200_attention_decode_noalloc(const s2p_bf16* q, const s2p_bf16* k_cache, const s2p_bf16* v_cache,
                                             s2p_bf16* out, int q_heads, int kv_heads, int head_dim, int pos,
                                             int max_seq, cudaStream_t stream);

/* ===== paged 4-bit cache (no counterpart in the reference, whose sessions own contiguous bf16 or INT8 planes) =====
 *
 * Keys and values of many sequences in pages of 64 positions, 4 bits a channel, with what writes them, what attends over
 * them and what moves their pages.  Sequences that begin alike (a voice's prompt) share pages instead of copying them.
 *
 * All state is the caller's, in device memory of the current device, and every call works in stream order on it without
 * reading anything back, so a captured graph of reserve, append and attention calls replays as the sequences grow.  Calls
 * that share a cache or a workspace must be ordered: on one stream, or by events.
 *
 * A pool is n_pages pages of s2p_b200_kv4_page_bytes() bytes: [layers][kv_heads][4 blocks of 16 positions][2560 bytes].
 * In groups of 32 channels of one position a code c (0..15) stands for s c + m, with f16 m = the group's smallest value and
 * f16 s = (largest - smallest) / 15 (each rounded to nearest), c = (x - m) / s rounded to the nearest, ties to even, kept in
 * 0..15 (0 where s is 0).  Values beyond +-65504 are kept at that, a NaN takes code 0, and a group of nothing but NaN stands for zeros.
 * Block of position p (p % 16 = i), byte offsets; channel d of group j = d / 32, e = d % 32; even d in the low four bits:
 *   keys    codes       64 i + 16 (e / 8) + 4 j + (e % 8) / 2
 *           s, m        2048 + 16 i + 2 j,  2056 + 16 i + 2 j
 *   values  codes       1024 + 512 (i / 8) + 64 (e / 4) + 16 (i / 2 % 4) + 8 (i % 2) + 2 j + (e % 4) / 2
 *           s, m        2304 + 16 (i / 2) + 4 j + 2 (i % 2),  2432 + the same
 * (the order in which the matrix instructions of the attention take them: a lane's bytes lie together). */
#define S2P_B200_KV4_PAGE 64
#define S2P_B200_KV4_MAX_BATCH 1024 /* sequences of one batch */
#define S2P_B200_KV4_MAX_LIST 256   /* sequences of one fork or release call */

typedef struct {
    void* pages;      /* the pool, 128-byte aligned */
    int32_t* table;   /* [max_seqs][table_stride]: page of positions 64 j .. 64 j + 63; an entry outside the pool (-1) holds nothing */
    int32_t* lens;    /* [max_seqs] positions held; table entries behind them are -1 */
    int32_t* refs;    /* [n_pages] table entries that name the page; 0 = free */
    void* work;       /* 256-byte aligned; zeroed once by the caller, before its first use; caches may share one */
    size_t work_bytes;
    int n_pages, layers, kv_heads, q_heads; /* up to 2^22 pages; q_heads a multiple of kv_heads, at most 16 times as many; width 128 */
    int max_seqs, table_stride;             /* table_stride up to 2^24 */
} s2p_b200_kv4;

/* The rows of a tick or a prompt slice: entry b brings rows row0[b] .. row0[b + 1] - 1 of the activations, at positions
 * pos0[b], pos0[b] + 1, ... of sequence seqs[b].  All arrays are device memory.  A sequence stands in a batch once; an entry
 * may have no rows; entries whose pos0 is negative or beyond 2^30, or whose sequence is outside 0 .. max_seqs - 1, store
 * nothing and see nothing, and zeros come out for their rows; rows behind row0[n] are left as they were. */
typedef struct {
    const int32_t* seqs; /* [n] */
    const int32_t* row0; /* [n + 1], not decreasing */
    int32_t* pos0;       /* [n], written by reserve */
    int n;
    int rows;     /* rows of the activations: those from row0[n] on are padding */
    int max_rows; /* the most rows that an entry has; only the choice of kernels goes by it, so it may be more or less */
} s2p_b200_kv4_batch;

size_t s2p_b200_kv4_page_bytes(int layers, int kv_heads);
/* workspace of every call on this cache, attention with batches of up to `rows` rows; 0 if the cache's sizes cannot be served */
size_t s2p_b200_kv4_work_bytes(const s2p_b200_kv4* c, int rows);
/* S2P_ERR_INTERNAL if a bounded wait of an attention call on this workspace gave up, once; rows of the calls since the status was last asked for may
 * be lost.  Waits for the stream (so not under capture). */
s2p_status s2p_b200_kv4_status(const s2p_b200_kv4* c, cudaStream_t stream);

/* Room for the batch's rows: pos0 = positions held, lens += rows, and free pages (lowest first, in the batch's order) for
 * what the last held page does not take.  An entry that needs more pages than all before it leave (those of refused ones count, so
 * that none goes ahead of them), or more table entries than there are, or whose sequence stands in the batch before it, is refused: pos0 = -1, and it keeps
 * what it held.  info (device, may be NULL): pages free afterwards, entries refused. */
s2p_status s2p_b200_kv4_reserve(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int32_t* info, cudaStream_t stream);

/* From raw rows qkv [rows, (q_heads + 2 kv_heads) * 128]: RMS norm of each query and key head (gains q_norm, k_norm [128];
 * NULL: no norm), rotation of its channel pairs (2 i, 2 i + 1) by position * rope_base^(-2 i / 128), queries to q
 * [rows, q_heads * 128], keys and values into the pages of `layer`.  In one pass and in 32 bits, the angle in 64: a query is
 * rounded once, to bf16, a key only to its 4 bits.  (s2pk_rope rounds cosine and sine to bf16, as the reference does.)
 * Rows whose position has no page come out in q all the same. */
s2p_status s2p_b200_kv4_append(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int layer, const s2p_bf16* qkv, const s2p_bf16* q_norm,
                               const s2p_bf16* k_norm, float eps, float rope_base, s2p_bf16* q, cudaStream_t stream);

/* out [rows, q_heads * 128]: softmax(q k / sqrt(128)) v over the positions of the row's sequence up to its own that have a
 * page; zeros where there is none.  out may be q.  Queries are below 2^100 in magnitude; a NaN or an infinity in a head's query
 * makes that head of the row NaN.  rows * kv_heads * table_stride is at most 2^29.  Scores, sums and results are in 32 bits; weights are rounded to
 * f16 for the products, and so are the weights times s in the kernel for tokens, keys and values s c + m in the one for slices; out is rounded to bf16.  That kernel's waits are bounded: see
 * s2p_b200_kv4_status.  Slices have it as long as the batch's work fits its list: rows / (2 (128 / group)) + 5 n up to about 4660, group = q_heads / kv_heads (one sequence up to
 * 298 thousand rows at four query heads to a kv head, 900 entries with 10 thousand).  Beyond that the kernel for tokens takes the whole batch, several times slower for long
 * slices: split such a batch. */
s2p_status s2p_b200_kv4_attention(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int layer, const s2p_bf16* q, s2p_bf16* out,
                                  cudaStream_t stream);

/* The values that the cache holds at the batch's positions, rounded to bf16: k and v [rows, kv_heads * 128], zeros where there is no page. */
s2p_status s2p_b200_kv4_read(const s2p_b200_kv4* c, const s2p_b200_kv4_batch* b, int layer, s2p_bf16* k, s2p_bf16* v, cudaStream_t stream);

/* Sequences children[i] become the first tokens[i] positions of parents[i] (fewer if it holds fewer; -1: all).  What the
 * children held is released first.  Full pages are shared; the last one, if it is not full, is copied into a free page
 * (lowest first, in the list's order), so that a shared page is never written again.  Without a free page child i is left
 * empty.  The lists are host memory, read before the call returns; a sequence stands among the children once and not among the
 * parents as well (S2P_ERR_INVALID).  info as above. */
s2p_status s2p_b200_kv4_fork(const s2p_b200_kv4* c, const int32_t* parents, const int32_t* children, const int32_t* tokens, int n,
                             int32_t* info, cudaStream_t stream);
/* Empties the sequences (host list, each once); pages that no other sequence holds become free. */
s2p_status s2p_b200_kv4_release(const s2p_b200_kv4* c, const int32_t* seqs, int n, cudaStream_t stream);
/* Moves pages until the used ones are the lowest: the k-th used page behind them to the k-th free one among them, with all
 * layers, references and table entries.  info: pages free, pages moved. */
s2p_status s2p_b200_kv4_compact(const s2p_b200_kv4* c, int32_t* info, cudaStream_t stream);

#pragma GCC visibility pop
#ifdef __cplusplus
}
#endif
#endif
