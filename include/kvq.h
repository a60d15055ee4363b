/*
 * kvq.h -- C ABI of libkvq.so, the MI355X (gfx950) INT8 KV-cache
 * decode-attention operator.
 *
 * Part 1 is the drop-in boundary: the exact extern "C" symbols of the
 * reference's kv_cache/ path (Murmurwkk/cuda-operators), with HIP types in
 * place of CUDA ones (hipSuccess == cudaSuccess == 0,
 * hipErrorInvalidValue == cudaErrorInvalidValue == 1).  One library exports
 * one `solve`; the reference's four kv_cache .cu files each export their own
 * and cannot be linked together.
 *
 * Part 2 is the extension the reference lacks (batch, grouped-query heads,
 * ragged lengths, sequence splits with a log-sum-exp merge, appending a
 * quantised token).  Each query head hq of batch b computes exactly the
 * reference's single-head math over kv head hq / (Hq/Hkv) and the first
 * lengths[b] tokens.
 *
 * Layouts (row-major, contiguous; all pointers are device pointers):
 *   reference ABI:  Q[H,d] fp32, K/V[H,N,d] int8, k/v_scale[H,N] fp32, out[H,d]
 *   extension:      q[B,Hq,d], k/v cache[B,Hkv,cap,d] int8,
 *                   k/v scale[B,Hkv,cap] fp32, out[B,Hq,d], lengths[B] int32
 *
 * Math (both parts): s_t = (sum_i q_i * K[t,i]) * k_scale[t] * softmax_scale,
 * p = softmax(s), out_i = sum_t p_t * (V[t,i] * v_scale[t]); softmax_scale
 * defaults to 1/sqrtf(d) as in the reference.
 */
#ifndef KVQ_H
#define KVQ_H

#include <stddef.h>
#include <stdint.h>

#include <hip/hip_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Largest head_dim any entry point but dense attention accepts (there: 1024).
 * Decode runs tuned kernels at 32 and multiples of 16 from 48 to 256, the
 * prefill quantiser at multiples of 4 (fp32) or 8 (bf16) up to 256,
 * kvq_quantize_rows_launch at 32, 64, 128 and 256, dense attention up to 256;
 * any other value up to the bound runs a generic kernel. */
#define KVQ_MAX_HEAD_DIM 4096

/* Longest sequence any decode entry point attends to, in tokens: seq_len of
 * the reference entry points, and the effective max_seq_len of the extension
 * (max_seq_len, or the capacity when it is 0).  The kernels count tokens and
 * tiles in 32-bit integers; beyond this bound the call is rejected with
 * hipErrorInvalidValue (solve: one stderr line).  Capacities and page tables
 * may be larger. */
#define KVQ_MAX_SEQ_LEN (1 << 30)

/* ===================== Part 1: reference entry points ===================== */

/* Replaces `solve`, kv_cache/KV_int8.cu:306-316 (also KV_int8_single_buffer.cu:260-270,
 * KV_int8_split_optimized.cu:294-304, new_kvint8.cu:102-104).
 * Legacy void ABI: invalid arguments print one line to stderr and return
 * without device work (as KV_int8_split_optimized.cu:306-324).  Runs
 * asynchronously on the null stream.  Split workspace comes from a per-device
 * cache owned by the library (allocated on first use, grown when needed). */
#ifndef KVQ_OMIT_DECODE_SOLVE /* defined by code that declares the attention `solve` (kvq_attention.h) */
void solve(const float* Q, const int8_t* K_int8, const int8_t* V_int8,
           const float* k_scale, const float* v_scale, float* output,
           int num_heads, int seq_len, int head_dim);
#endif

/* Replaces `kv_int8_split_launch`, kv_cache/KV_int8_split_optimized.cu:266-292.
 * S is caller-owned scratch of at least num_heads*seq_len floats; it holds the
 * per-split partial (max, sum, acc[d]) records, so at most seq_len/(head_dim+2)
 * splits per head are used (1 split needs no scratch at all).
 * Returns hipErrorInvalidValue, before any HIP call, for a null pointer,
 * num_heads/seq_len/head_dim <= 0, head_dim > KVQ_MAX_HEAD_DIM or
 * seq_len > KVQ_MAX_SEQ_LEN; otherwise the launch status.  Asynchronous on `stream`; the caller checks completion. */
hipError_t kv_int8_split_launch(const float* Q, const int8_t* K_int8, const int8_t* V_int8,
                                const float* k_scale, const float* v_scale, float* output,
                                int num_heads, int seq_len, int head_dim, float* S,
                                hipStream_t stream);

/* Replaces `kv_int8_simple_launch`, kv_cache/new_kvint8.cu:83-100 (identical
 * signature and contract to kv_int8_split_launch; same kernels here). */
hipError_t kv_int8_simple_launch(const float* Q, const int8_t* K_int8, const int8_t* V_int8,
                                 const float* k_scale, const float* v_scale, float* output,
                                 int num_heads, int seq_len, int head_dim, float* S,
                                 hipStream_t stream);

/* ============== Part 2: extension (no counterpart in the reference) ============== */

typedef struct kvq_decode_params {
    int batch;             /* B  >= 1 */
    int num_q_heads;       /* Hq >= 1, a multiple of num_kv_heads */
    int num_kv_heads;      /* Hkv >= 1 */
    int head_dim;          /* d in [1, KVQ_MAX_HEAD_DIM] */
    int capacity;          /* token stride of one (b, kv_head) cache row block, >= 1 */
    int max_seq_len;       /* uniform length when lengths == NULL; otherwise an upper
                              bound on every lengths[b] (0 means capacity) */
    const int32_t* lengths;/* device [B] or NULL; each clamped on device to
                              [0, max_seq_len] (max_seq_len 0: capacity);
                              a sequence of length 0 yields a zero output row */
    const float* q;        /* [B, Hq, d] */
    int8_t* k_cache;       /* [B, Hkv, capacity, d]; written only by a fused append */
    int8_t* v_cache;
    float* k_scale;        /* [B, Hkv, capacity] */
    float* v_scale;
    float* out;            /* [B, Hq, d], fully overwritten */
    float softmax_scale;   /* <= 0 selects 1/sqrtf(d) */
    int num_splits;        /* 0 = choose; otherwise the split count per sequence (the
                              tuned kernels round chunks up to whole tiles, so fewer
                              splits may run) */
    /* Fused append (both NULL = off).  When set, token length_b - 1 of every
     * (b, kv_head) is first quantised from k_new/v_new [B, Hkv, d] fp32 into the
     * cache (int8 values + scale, the same bits as kvq_append_launch), then
     * attended over; the caller's lengths already count the new token.  This
     * holds for every sequence: one that has no new token in this step is given
     * length 0, or its last token is overwritten. */
    const float* k_new;
    const float* v_new;
} kvq_decode_params;

/* Bytes of workspace kvq_decode_launch needs for `p` (0 when one split
 * suffices).  The workspace holds per-split partials and one arrival counter
 * per (b, kv_head, head group); it must be zero-filled once after allocation
 * (kvq_workspace_init) and is left zeroed by every completed launch.  Calls
 * that overlap in time must not share a workspace. */
size_t kvq_decode_workspace_size(const kvq_decode_params* p);

/* Zero-fills a workspace on `stream` with a fill kernel (no hipMemset). */
hipError_t kvq_workspace_init(void* workspace, size_t workspace_bytes, hipStream_t stream);

/* Decode attention (plus the optional fused append) in one kernel launch:
 * splits write partial (max, sum, acc) records and the last split of each
 * sequence to finish merges them with a log-sum-exp reduction.
 * Returns hipErrorInvalidValue before any HIP call on a bad argument or a
 * workspace smaller than kvq_decode_workspace_size(p). */
hipError_t kvq_decode_launch(const kvq_decode_params* p, void* workspace, size_t workspace_bytes,
                             hipStream_t stream);

/* Size of the fixed device scratch array of kvq_decode_launch_noalloc. */
#define KVQ_NOALLOC_SCRATCH_BYTES (16u << 20)

/* No counterpart in the reference.  kvq_decode_launch without a workspace
 * argument and without any allocation, for callers that cannot allocate device
 * memory (code under graph capture, tight serving loops, harnesses that forbid
 * hipMalloc).  The split records and arrival counters live in a fixed
 * KVQ_NOALLOC_SCRATCH_BYTES device array that each GPU holds until the process
 * ends (its counters are zero-filled by a kernel on the first call on each
 * device and left at zero by every completed launch).  Same plan, kernels and
 * result bits as kvq_decode_launch while kvq_decode_workspace_size(p) is at most
 * KVQ_NOALLOC_SCRATCH_BYTES.  Beyond that the call is planned again without
 * padded tiles (which can need records where other kernels need none: other
 * kernels and summation order, the same results to rounding);
 * hipErrorInvalidValue when that plan does not fit either, and for the
 * arguments kvq_decode_launch rejects.  All calls on one GPU share the array: calls that
 * overlap in time on one GPU (different streams, or host threads) race. */
hipError_t kvq_decode_launch_noalloc(const kvq_decode_params* p, hipStream_t stream);

typedef struct kvq_append_params {
    int batch, num_kv_heads, head_dim, capacity;
    const int32_t* positions; /* device [B] write position per sequence, or NULL */
    int uniform_position;     /* used when positions == NULL */
    const float* k_new;       /* [B, Hkv, d] fp32 */
    const float* v_new;
    int8_t* k_cache;          /* [B, Hkv, capacity, d] */
    int8_t* v_cache;
    float* k_scale;           /* [B, Hkv, capacity] */
    float* v_scale;
} kvq_append_params;

/* Quantises one new K and V token per (b, kv_head): scale = max|x|/127.0f
 * (IEEE division), q = clamp(rintf(x/scale), -127, 127); a zero (or
 * underflowing) scale stores 0 and all-zero int8.  Positions outside
 * [0, capacity) are skipped.  lengths are not modified. */
hipError_t kvq_append_launch(const kvq_append_params* p, hipStream_t stream);

/* Bulk (prefill) quantiser: x[rows, d] fp32 -> q[rows, d] int8 + scale[rows],
 * the same per-row rule as kvq_append_launch. */
hipError_t kvq_quantize_rows_launch(const float* x, int64_t rows, int head_dim, int8_t* q,
                                    float* scale, hipStream_t stream);

/* ============ Part 3: paged KV cache (no counterpart in the reference) ============
 *
 * The cache lives in a pool of pages instead of one contiguous row block per
 * (b, kv_head):
 *   k/v_pages        [num_pages, Hkv, page_size, d] int8
 *   k/v_scale_pages  [num_pages, Hkv, page_size]    fp32
 *   block_table      [batch, max_pages_per_seq]     int32 page ids
 * Token t of sequence b is slot t % page_size of page
 * block_table[b * max_pages_per_seq + t / page_size]; within a page each kv
 * head's page_size rows are contiguous (page_size * d bytes).  Page ids
 * outside [0, num_pages) are clamped into it on the device (no fault; the
 * result is then meaningless).  Everything else -- math, lengths, splits,
 * fused append, workspace rules -- is as for kvq_decode_params, and a paged
 * cache holding the same tokens gives the same output. */

typedef struct kvq_paged_decode_params {
    int batch;              /* B >= 1 */
    int num_q_heads;        /* Hq >= 1, a multiple of num_kv_heads */
    int num_kv_heads;       /* Hkv >= 1 */
    int head_dim;           /* d in [1, KVQ_MAX_HEAD_DIM] */
    int page_size;          /* tokens per page, >= 1 (a multiple of 16 runs the tuned kernels) */
    int num_pages;          /* pages in the pool, >= 1 */
    int max_pages_per_seq;  /* row stride of block_table, >= 1 */
    int max_seq_len;        /* uniform length when lengths == NULL; otherwise a bound on
                               every lengths[b] (0: max_pages_per_seq * page_size) */
    const int32_t* block_table; /* device [B, max_pages_per_seq] */
    const int32_t* lengths; /* device [B] or NULL; clamped on device to [0, max_seq_len] */
    const float* q;         /* [B, Hq, d] */
    int8_t* k_pages;        /* [num_pages, Hkv, page_size, d]; written only by a fused append */
    int8_t* v_pages;
    float* k_scale_pages;   /* [num_pages, Hkv, page_size] */
    float* v_scale_pages;
    float* out;             /* [B, Hq, d], fully overwritten */
    float softmax_scale;    /* <= 0 selects 1/sqrtf(d) */
    int num_splits;         /* 0 = choose; otherwise the split count per sequence */
    const float* k_new;     /* fused append as in kvq_decode_params (both NULL = off) */
    const float* v_new;
} kvq_paged_decode_params;

/* Workspace bytes for kvq_paged_decode_launch (same rules as
 * kvq_decode_workspace_size). */
size_t kvq_paged_decode_workspace_size(const kvq_paged_decode_params* p);

/* Decode attention over a paged cache, plus the optional fused append.
 * Returns hipErrorInvalidValue before any HIP call on a bad argument or a
 * workspace smaller than kvq_paged_decode_workspace_size(p). */
hipError_t kvq_paged_decode_launch(const kvq_paged_decode_params* p, void* workspace,
                                   size_t workspace_bytes, hipStream_t stream);

typedef struct kvq_paged_append_params {
    int batch, num_kv_heads, head_dim, page_size, num_pages, max_pages_per_seq;
    const int32_t* block_table; /* device [B, max_pages_per_seq] */
    const int32_t* positions;   /* device [B] token position per sequence, or NULL */
    int uniform_position;       /* used when positions == NULL */
    const float* k_new;         /* [B, Hkv, d] fp32 */
    const float* v_new;
    int8_t* k_pages;            /* [num_pages, Hkv, page_size, d] */
    int8_t* v_pages;
    float* k_scale_pages;       /* [num_pages, Hkv, page_size] */
    float* v_scale_pages;
} kvq_paged_append_params;

/* kvq_append_launch for a paged cache: the token goes to its position's page
 * slot; positions outside [0, max_pages_per_seq * page_size) are skipped. */
hipError_t kvq_paged_append_launch(const kvq_paged_append_params* p, hipStream_t stream);

/* ============ Part 4: prefill quantiser (no counterpart in the reference) ============
 *
 * Writes L new tokens per (b, kv head) into a contiguous or paged cache:
 * K and V rows x[B, Hkv, L, d] (fp32 or bf16) are quantised with the rule of
 * kvq_append_launch and stored at token positions start_b .. start_b + L - 1
 * (start_b = start[b], or uniform_start when start is NULL).  Positions
 * outside [0, capacity) -- paged: [0, max_pages_per_seq * page_size) -- are
 * skipped.  bf16 inputs are widened to fp32 exactly before the same rule. */

#define KVQ_DTYPE_F32 0
#define KVQ_DTYPE_BF16 1

typedef struct kvq_prefill_params {
    int batch, num_kv_heads, head_dim;
    int tokens;               /* L >= 0 new tokens per (b, kv head) */
    int dtype;                /* KVQ_DTYPE_F32 or KVQ_DTYPE_BF16 */
    const void* k_new;        /* [B, Hkv, L, d] */
    const void* v_new;
    const int32_t* start;     /* device [B] first position per sequence, or NULL */
    int uniform_start;        /* used when start == NULL */
    int capacity;             /* contiguous cache: tokens per (b, kv head) row block */
    int8_t* k_cache;          /* contiguous [B, Hkv, capacity, d] or pages [num_pages, Hkv, page_size, d] */
    int8_t* v_cache;
    float* k_scale;           /* [B, Hkv, capacity] or [num_pages, Hkv, page_size] */
    float* v_scale;
    const int32_t* block_table; /* NULL: contiguous cache; else paged (as kvq_paged_decode_params) */
    int page_size, num_pages, max_pages_per_seq;
} kvq_prefill_params;

/* One launch quantises all B*Hkv*L K and V rows. */
hipError_t kvq_prefill_quantize_launch(const kvq_prefill_params* p, hipStream_t stream);

/* ============ Part 5: dense fp32 attention (prefill-shaped) ============
 *
 * out[M, d] = softmax(Q K^T * scale) V for Q[M, d], K/V[N, d] fp32, one head,
 * no mask; the operator of attention/softmax_new.cu:87-281.  Inputs must be
 * finite (as the reference requires, attention/softmax_new.cu:237). */

/* Replaces attention_online_launch (attention/softmax_new.cu:239-281): same
 * arguments, scale 1/sqrtf(d), hipErrorInvalidValue for a NULL pointer,
 * M, N or d <= 0, or d > 1024 (the reference's limit, :252).  When the
 * queries alone cannot fill the GPU the keys are split over workgroups; the
 * partial results then live in a workspace the library owns, one per (device,
 * stream), allocated on first use and grown on demand (hipMalloc).  Callers
 * that must not allocate use kvq_attention_launch with their own workspace.
 * The reference's compatibility `solve(Q, K, V, output, M, N, d)`
 * (attention/softmax_new.cu:283-287) is not exported: its symbol is the
 * decode `solve` above. */
hipError_t attention_online_launch(const float* Q, const float* K, const float* V, float* output, int M, int N,
                                   int d, hipStream_t stream);

typedef struct kvq_attention_params {
    int M, N, d;              /* queries, keys, head dim (1 <= d <= 1024) */
    const float* q;           /* [M, d] */
    const float* k;           /* [N, d] */
    const float* v;           /* [N, d] */
    float* out;               /* [M, d] */
    float softmax_scale;      /* 0 -> 1/sqrtf(d) */
    int num_splits;           /* 0 -> chosen by the library; else a request (clamped) */
} kvq_attention_params;

/* Workspace bytes kvq_attention_launch needs for p (0: none, or invalid p):
 * the split records, which need no initial contents. */
size_t kvq_attention_workspace_size(const kvq_attention_params* p);

/* attention_online_launch with an explicit scale, split request and
 * caller-owned workspace (16-byte aligned, at least
 * kvq_attention_workspace_size(p) bytes); allocates nothing.  With splits, a
 * second kernel merges the records.  Launches that share a workspace must be
 * ordered (one stream).  hipErrorInvalidValue, before any HIP call, for the
 * checks of attention_online_launch, M or N above INT_MAX - 1024, a negative
 * num_splits, or a workspace too small, NULL or misaligned when one is
 * needed.  At head dims other than 32, 64, 128 and 256 the keys are split only
 * on request, and a request with a NULL workspace runs unsplit. */
hipError_t kvq_attention_launch(const kvq_attention_params* p, void* workspace, size_t workspace_bytes,
                                hipStream_t stream);

/* Library version string, e.g. "kvq 0.1.0 gfx950". */
const char* kvq_version(void);

/* ============ Part 6: plan queries and diagnostics (no counterpart in the reference) ============
 *
 * Host-only: these read no device memory and make no HIP call, so pointers
 * may be any values with the alignment of the real ones.  They report what
 * the matching launch would do. */

#define KVQ_KERNEL_DECODE_GENERIC 0   /* decode_generic: any head dim or alignment */
#define KVQ_KERNEL_DECODE_VALU 1      /* decode_fast: per-lane FMAs; head dim 32 and multiples of 16
                                         from 48 to 256 (between the powers of two with padded lanes) */
#define KVQ_KERNEL_DECODE_MFMA 2      /* decode_mfma: grouped-query heads on matrix cores */
#define KVQ_KERNEL_ATTENTION_MFMA 3   /* attention_limbs: query blocks on matrix cores, d <= 256 */
#define KVQ_KERNEL_ATTENTION_ROWS 4   /* attention_rows: up to 8 queries per workgroup */
#define KVQ_KERNEL_ATTENTION_GENERIC 5 /* attention_generic: any head dim or alignment */
#define KVQ_KERNEL_ATTENTION_DIRECT 6  /* attention_direct: 9-64 queries, 16 per wave, no LDS tiles */

#define KVQ_SPLITS_STATIC 0     /* splits and chunk fixed on the host */
#define KVQ_SPLITS_IN_KERNEL 1  /* ragged batch planned inside the decode kernel */
#define KVQ_SPLITS_SCHEDULE 2   /* ragged batch planned by a schedule launch */
#define KVQ_SPLITS_TILES 3      /* ragged batch as one tile stream, split evenly over the
                                   matrix-core kernel's waves inside the kernel */

typedef struct kvq_plan_info {
    int kernel;             /* KVQ_KERNEL_* */
    int heads_per_group;    /* query heads one workgroup computes */
    int splits;             /* static plans: splits per sequence (1 = unsplit); 0 otherwise */
    int chunk;              /* static plans: tokens (keys) per split */
    int split_plan;         /* KVQ_SPLITS_* */
    int query_block;        /* attention: queries per workgroup; decode: 0 */
    size_t workspace_bytes; /* workspace (or scratch S) bytes the launch uses */
    int tile_tokens;        /* decode: tokens one workgroup iteration of the tuned kernel covers
                               (0: generic kernel); attention: 0 */
} kvq_plan_info;

/* The plan of kv_int8_split_launch / kv_int8_simple_launch for these
 * arguments; workspace_bytes is the part of S it uses (<= 4*num_heads*seq_len).
 * hipErrorInvalidValue for arguments the launch rejects. */
hipError_t kvq_reference_plan(const float* Q, const int8_t* K_int8, const int8_t* V_int8, int num_heads,
                              int seq_len, int head_dim, kvq_plan_info* info);
/* The plan of kvq_decode_launch for p. */
hipError_t kvq_decode_plan(const kvq_decode_params* p, kvq_plan_info* info);
/* The plan of kvq_paged_decode_launch for p. */
hipError_t kvq_paged_decode_plan(const kvq_paged_decode_params* p, kvq_plan_info* info);
/* The plan of kvq_attention_launch for p and a workspace of that size; also
 * that of attention_online_launch (p with softmax_scale 0 and num_splits 0),
 * except that with its own workspace it splits the keys at every head dim up to
 * 256, and where this plan needs no workspace because 128-query blocks fill the
 * GPU (32641 queries at d = 128). */
hipError_t kvq_attention_plan(const kvq_attention_params* p, kvq_plan_info* info);

/* Diagnostic switches in force, read once from the environment:
 * bit 0: KVQ_DEBUG_SYNC ("1", "true", "yes" or "on"): every launching entry
 *        point synchronises its stream after its launches and returns the first
 *        error (not while the stream is being captured);
 * bits 4-7: KVQ_FORCE_KERNEL: 1 = "valu" (decode plans avoid the matrix-core
 *        kernel), 2 = "generic" (decode plans avoid both tuned kernels). */
int kvq_diagnostics(void);

/* ============ Part 7: a paged cache's life on the GPU (no counterpart in the reference) ============
 *
 * What a serving loop does around paged decode, without host round trips:
 *   kvq_page_map_launch       block tables, free pages and slots from request lengths
 *   kvq_slot_write_launch     a packed (ragged) batch of K/V rows quantised into its slots
 *   kvq_slot_read_launch      cached tokens as fp32 or bf16 rows
 *   kvq_page_bounds_launch    int8 bounds of each page's keys
 *   kvq_sparse_decode_launch  a decode step over the pages that the bounds rank highest
 * A slot is a token's place in the pool: page id * page_size + its place in the
 * page; pool layouts and block tables are those of part 3.  Every entry point
 * returns hipErrorInvalidValue before any HIP call on a bad argument, is
 * asynchronous on `stream`, allocates nothing and can be captured. */

/* Most sequences of one page map. */
#define KVQ_PAGE_MAP_MAX_BATCH 4096

typedef struct kvq_page_map_params {
    int batch;               /* B in [1, KVQ_PAGE_MAP_MAX_BATCH] */
    int page_size;           /* tokens per page, >= 1 */
    int num_pages;           /* pages in the pool; num_pages * page_size <= INT_MAX */
    int max_pages_per_seq;   /* row stride of block_table; a sequence holds at most
                                max_pages_per_seq * page_size tokens */
    int max_tokens;          /* T >= 0: rows of the packed batch */
    const int32_t* new_tokens; /* device [B]: tokens to add; negative: to take off the end */
    const int32_t* lengths;  /* device [B]: tokens held, each clamped to [0, capacity] */
    int32_t* block_table;    /* device [B, max_pages_per_seq], updated in place */
    int32_t* free_pages;     /* device [num_pages]: the free stack, updated in place */
    const int32_t* free_count; /* device [1]: its entries, clamped to [0, num_pages] */
    int32_t* new_lengths;    /* device [B]; may be `lengths` */
    int32_t* new_free_count; /* device [1]; may be `free_count` */
    int32_t* granted;        /* device [B]: tokens added (taken off: negative; refused: 0) */
    int32_t* token_offsets;  /* device [B + 1]: first packed row of each sequence, then the rows' number */
    int32_t* slot_map;       /* device [T]: slot of each packed row, or NULL */
    int32_t* token_seq;      /* device [T]: its sequence, or NULL */
    int32_t* token_pos;      /* device [T]: its position in the sequence, or NULL */
} kvq_page_map_params;

/* Grows and shrinks the sequences of a paged cache.
 * - Sequence b asks for max(new_tokens[b], 0) packed rows, which follow those of
 *   the sequences before it; offsets saturate at max_tokens.
 * - A request is granted whole or refused whole (length, table and pages stay).
 *   It is refused when it does not fit block_table's row or the packed rows;
 *   and, if it needs a page, when the pages that it and the sequences before it
 *   need (those refused for want of pages among them) are more than there are.
 * - Sequences that shrink give up the pages behind their new end first: these go
 *   onto the free stack in the order (sequence, page), so the same call can hand
 *   them out.  The i-th page that growing sequences take, in that order, is the
 *   i-th from the stack's top.  Entries behind the end of the stack, and table
 *   entries behind a sequence's last page, have no meaning and are left as they
 *   were.
 * - slot_map, token_seq and token_pos are wholly written: a refused request's
 *   rows have slot -1; rows behind the last have -1 in all three.  A row whose
 *   page id lies outside the pool has slot -1.
 * - Pages belong to one sequence; a page in two tables is given up twice.
 * - A decode step's fused append (k_new, v_new) writes token length_b - 1 of every
 *   sequence, granted or not: of one that was refused, waits or shrank that is a
 *   token it holds.  Rows written through slot_map skip those sequences; a step
 *   with a fused append is given length 0 for them (where granted[b] <= 0).
 * Workspace: kvq_page_map_workspace_size bytes (0 for small batches), zero-filled
 * once (kvq_workspace_init) and left zeroed.  Calls on one pool must be ordered. */
size_t kvq_page_map_workspace_size(const kvq_page_map_params* p);
hipError_t kvq_page_map_launch(const kvq_page_map_params* p, void* workspace, size_t workspace_bytes,
                               hipStream_t stream);

typedef struct kvq_slot_write_params {
    int tokens;               /* T >= 0 packed rows; T * num_kv_heads < 2^31 */
    int num_kv_heads, head_dim;
    int page_size, num_pages; /* num_pages * page_size <= INT_MAX */
    int dtype;                /* KVQ_DTYPE_F32 or KVQ_DTYPE_BF16 */
    const void* k_new;        /* [T, Hkv, d]: a token's heads lie together */
    const void* v_new;
    int64_t k_stride;         /* elements from a token to the next, >= Hkv * d (0: Hkv * d) */
    int64_t v_stride;
    const int32_t* slots;     /* device [T]; a slot outside the pool skips its row */
    int8_t* k_pages;          /* [num_pages, Hkv, page_size, d] */
    int8_t* v_pages;
    float* k_scale_pages;     /* [num_pages, Hkv, page_size] */
    float* v_scale_pages;
} kvq_slot_write_params;

/* The quantiser of kvq_append_launch (same bits) over a packed batch.  Slots
 * must be distinct: a slot that is named twice holds some mixture of its rows. */
hipError_t kvq_slot_write_launch(const kvq_slot_write_params* p, hipStream_t stream);

typedef struct kvq_slot_read_params {
    int tokens;               /* T >= 0; T * num_kv_heads < 2^31 */
    int num_kv_heads, head_dim;
    int page_size, num_pages; /* num_pages * page_size <= INT_MAX */
    int dtype;                /* of the outputs: KVQ_DTYPE_F32 or KVQ_DTYPE_BF16 */
    const int32_t* slots;     /* device [T], in any order and number */
    const int8_t* k_pages;    /* [num_pages, Hkv, page_size, d] */
    const int8_t* v_pages;
    const float* k_scale_pages;
    const float* v_scale_pages;
    void* k_out;              /* row (t, h) at t * token_stride + h * head_stride, wholly written */
    void* v_out;
    int64_t token_stride;     /* elements, for both outputs; [T, Hkv, d]: Hkv * d, d; */
    int64_t head_stride;      /* [Hkv, T, d]: d, T * d.  Rows must not overlap */
} kvq_slot_read_params;

/* Cached rows as numbers: code * scale in fp32, rounded to nearest even for
 * bf16; a slot outside the pool gives a zero row. */
hipError_t kvq_slot_read_launch(const kvq_slot_read_params* p, hipStream_t stream);

typedef struct kvq_page_bounds_params {
    int batch, num_kv_heads, head_dim; /* batch < 2^24 */
    int page_size, num_pages, max_pages_per_seq; /* max_pages_per_seq * num_kv_heads must fit an int */
    int max_seq_len;            /* as kvq_paged_decode_params */
    const int32_t* block_table; /* device [B, max_pages_per_seq] */
    const int32_t* start;       /* device [B]: first token whose page is to be done (clamped at 0), or NULL: 0 */
    const int32_t* lengths;     /* device [B] or NULL; clamped on device to [0, max_seq_len] */
    const int8_t* k_pages;      /* [num_pages, Hkv, page_size, d] */
    const float* k_scale_pages; /* [num_pages, Hkv, page_size] */
    int8_t* bounds;             /* [num_pages, Hkv, 2, d]: highs, then lows */
    float* bound_scale;         /* [num_pages, Hkv] */
} kvq_page_bounds_params;

/* Bounds of the keys of every page that holds a token in [start_b, length_b),
 * over its tokens below length_b: with s_t the tokens' scales and k_t their
 * codes, S = max |s_t|, highs ceil(max_t k_t r_t) and lows floor(min_t k_t r_t)
 * per dim for r_t = s_t / S (quotient and product rounded in fp32), so every key
 * lies in S * [low, high] but for those roundings.  S = 0: bounds 0.  S not
 * finite: bounds 127 and -127 under the scale +inf, which rank first.  Codes lie
 * in [-127, 127], as every quantiser here writes them.  A page in two tables must
 * hold the same tokens below both lengths. */
hipError_t kvq_page_bounds_launch(const kvq_page_bounds_params* p, hipStream_t stream);

typedef struct kvq_sparse_decode_params {
    kvq_paged_decode_params decode; /* the dense step: attends to at most max_selected pages of it */
    int max_selected;         /* pages per (sequence, kv head), >= keep_first + keep_last */
    int keep_first;           /* leading pages attended whatever their score, >= 0 */
    int keep_last;            /* trailing pages, >= 1 */
    int8_t* bounds;           /* [num_pages, Hkv, 2, d], as kvq_page_bounds_launch writes them */
    float* bound_scale;       /* [num_pages, Hkv] */
    int32_t* selected;        /* [B, Hkv, max_selected] out: page id * Hkv + kv head of the pages attended,
                                 ascending in the sequence, then -1 */
    int32_t* selected_lengths;/* [B, Hkv] out: tokens in them */
} kvq_sparse_decode_params;

/* Decode attention over the pages of each sequence that rank highest for the
 * query, per kv head.  A sequence of at most max_selected pages is attended
 * whole (as kvq_paged_decode_launch does).  Of a longer one, keep_first leading
 * and keep_last trailing pages, and of the others those with the highest scores,
 * equal ones in page order.
 * Score of a page, for the G query heads of a kv head: the heads' q are quantised
 * with one scale (max |q| over all of them / 127, the rule of kvq_append_launch);
 * score = float(max over heads of sum_i max(q_i high_i, q_i low_i)) * bound_scale,
 * an exact integer with two fp32 roundings, so every implementation ranks alike.
 * A NaN score ranks first.
 * Bounds: of every page but the last keep_last they must be current.  When the
 * step's token opens a page (length_b - 1 is a multiple of page_size), the page
 * before it has become whole and its bounds are written by this call; so decode
 * steps of one token keep them current, while tokens written otherwise need
 * kvq_page_bounds_launch.
 * `selected` is a block table of the pool seen as num_pages * Hkv pages of one kv
 * head ([num_pages * Hkv, 1, page_size, d]), for batch * Hkv sequences of
 * selected_lengths tokens.
 * Workspace as for kvq_paged_decode_launch: kvq_sparse_decode_workspace_size
 * bytes, zero-filled once, left ready by every completed launch.  num_pages * Hkv
 * and B * Hkv * max_selected must fit an int, and B * Hkv must be below 2^23. */
size_t kvq_sparse_decode_workspace_size(const kvq_sparse_decode_params* p);
hipError_t kvq_sparse_decode_launch(const kvq_sparse_decode_params* p, void* workspace, size_t workspace_bytes,
                                    hipStream_t stream);
/* The plan of the attention over the selected pages; workspace_bytes is the
 * whole call's.  Host-only (as part 6). */
hipError_t kvq_sparse_decode_plan(const kvq_sparse_decode_params* p, kvq_plan_info* info);

#ifdef __cplusplus
}
#endif

#endif /* KVQ_H */
