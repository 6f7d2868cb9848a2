/*
 * gfa.h - C ABI of the MI355X (gfx950) GQA flash-attention engine.
 *
 * Plain C: raw device pointers, element strides and sizes, a hipStream_t passed as
 * void*. No framework types cross this boundary. The library never allocates, frees
 * or synchronises; every call is stream-ordered on the caller's stream and device.
 *
 * Tensor layout: q/o/do/dq are (B, Hq, N, D); k/v/dk/dv are (B, Hkv, N, D); every
 * tensor is addressed through its own (batch, head, row) element strides and must have
 * a unit-stride head dimension and 16-byte aligned rows. lse/delta are float32
 * (B, Hq, lse_ld) with lse_ld >= GFA_LSE_LD(N): the backward kernels read whole query
 * tiles of up to 64 rows, so rows N..lse_ld-1 must exist (their values are never used).
 * Query head h reads KV head h / (Hq / Hkv) (contiguous groups). head_dim is 64, 128, 256
 * or 512 (the reference documents 64-512, powers of two); anything else returns
 * GFA_ERR_UNSUPPORTED, as does a (batch, head) slice that, with 127 rows of margin past its
 * end, spans more than 4 GiB.
 *
 * Variable-length and padded batches: seg_lo / seg_hi (optional, both or neither) are
 * int32 (B, N) tables, row b at seg_lo + b * N. Token t of row b attends, and is attended
 * by, only the tokens of keys [seg_lo[t], seg_hi[t]), intersected with the causal / window
 * rule. Each row must partition [0, N) into consecutive runs: a segment, whose tokens all
 * carry lo = first token and hi = one past its last, or padding, where token t carries
 * lo = hi = t (an empty segment: its O row is 0, its LSE -inf, and its dQ/dK/dV rows 0).
 * So both columns are non-decreasing. Left and right padding and packed sequences (the
 * reference's unsupported varlen case, README.md:255-262) are all such tables. The kernels
 * clamp table values to [0, N], so no content makes them address outside the tensors.
 *
 * The entry points replace the reference's Triton launch sites (file:line in
 * /root/reference, zzhhjjj/gemma-triton-flash-attn):
 *   gfa_fwd          flash_attn/attention.py:1454-1468 (_flash_attn_gqa_kernel launch,
 *                    STORE_LSE=True, training forward) and attention.py:589-601
 *                    (inference forward, STORE_LSE=False -> lse == NULL)
 *   gfa_bwd          flash_attn/attention.py:1506-1620 (dQ kernel with fused delta,
 *                    then the pack-GQA dKV kernel with its Q_SPLITS partial sums)
 *   gfa_config       the HEAD_DIM-keyed tile tables at attention.py:561-579, 1445-1451,
 *                    1498-1504, 1536-1564 and the Q_SPLITS choice at 1576-1587
 *   gfa_bwd_workspace_size
 *                    sizing of the (2,)+k.shape pre-zeroed buffer of attention.py:1594-1600
 *                    (here: fp32 partials, owned by the caller)
 */
#ifndef GFA_H_
#define GFA_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* The argument structs grow at their ends from version to version: a caller is compiled against the header of the library that it loads
 * (gfa_version() tells), sets every struct to zero first and then what it uses. */
#define GFA_VERSION 109 /* 1.0.9: requests that share blocks, drafted tokens; gfa_kv4_attn_args ends with shared_skip to shared_apart (1.0.8: key/value cache in 4 bits, 1.0.7: segment tables from position ids and masks, 1.0.6: materialised backward, 1.0.5: run-time work distribution, 1.0.4: attention dropout, 1.0.3: soft-capping) */

typedef enum {
  GFA_DTYPE_FP16 = 0,
  GFA_DTYPE_BF16 = 1
} gfa_dtype;

typedef enum {
  GFA_OK = 0,
  GFA_ERR_INVALID_ARGUMENT = 1, /* shape / stride / dtype / alignment / head-dim problem */
  GFA_ERR_UNSUPPORTED = 2,      /* valid request outside the built kernel set          */
  GFA_ERR_WORKSPACE = 3,        /* workspace missing or too small                      */
  GFA_ERR_LAUNCH = 4            /* the HIP runtime rejected a kernel launch            */
} gfa_status;

/* Smallest legal lse_ld for a sequence length. */
#define GFA_LSE_LD(seq_len) ((((seq_len) + 63) / 64) * 64)

/* gfa_bwd_args.stages bits */
#define GFA_BWD_DQ 1  /* recomputing form: delta + dQ kernel; materialised: dQ from the dS store */
#define GFA_BWD_DKV 2 /* dK/dV kernel (+ Q-split reduction); materialised: delta kernel, then dK/dV */

/* Element strides (batch, head, row) of one 4-D tensor; the head-dim stride is 1. */
typedef struct {
  int64_t batch, head, row;
} gfa_strides;

typedef struct {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  float* lse; /* (B, Hq, lse_ld) natural-log logsumexp; NULL = inference (not stored) */
  gfa_strides q_strides, k_strides, v_strides, o_strides;
  int32_t batch, heads_q, heads_kv, seq_len, head_dim;
  int32_t causal;      /* 0 / 1 */
  int32_t window;      /* sliding window; 0 = off; honoured only when causal; >= seq_len -> off */
  float scale;         /* softmax scale, finite and > 0; the reference uses 1/sqrt(head_dim) */
  int32_t dtype;       /* gfa_dtype, shared by q/k/v/o */
  int32_t block_kv;    /* 0 = library's choice (the registry's tile; small grids run a kernel that
                          splits the keys over a workgroup's waves), else a built tile width */
  int32_t lse_ld;      /* row length of lse (>= GFA_LSE_LD(seq_len)); ignored when lse == NULL */
  void* stream;        /* hipStream_t */
  const int32_t* seg_lo; /* optional (B, N) segment table (see above); NULL = one segment per row */
  const int32_t* seg_hi;
  float softcap;       /* 0 = off; > 0: every scaled score x = scale q.k becomes softcap tanh(x / softcap)
                          before the mask and softmax (transformers' logit soft-capping; the reference
                          has none). Runs the registry's default tiles (block_kv must be 0 or it). */
  float dropout_p;     /* 0 = off; in (0, 1): each P_ij is kept with probability 1 - dropout_p and scaled by
                          1 / (1 - dropout_p), else zeroed (the LSE is that of the undropped P). The mask
                          is a pure function of (dropout_seed, b, query head, i, j); the backward must get
                          the same seed. Not combined with softcap. Default tiles only, as softcap. */
  uint64_t dropout_seed;
} gfa_fwd_args;

typedef struct {
  const void* q;
  const void* k;
  const void* v;
  const void* o;
  const void* dout;
  const float* lse; /* from gfa_fwd, (B, Hq, lse_ld) */
  float* delta;     /* (B, Hq, lse_ld) scratch written by the dQ kernel: rowsum(dO * O), for
                       every row below seq_len rounded up to 32 (rows past seq_len repeat
                       row seq_len-1) */
  void* dq;
  void* dk;
  void* dv;
  gfa_strides q_strides, k_strides, v_strides, o_strides, do_strides, dq_strides, dk_strides, dv_strides;
  int32_t batch, heads_q, heads_kv, seq_len, head_dim;
  int32_t causal, window;
  float scale;
  int32_t dtype;
  int32_t q_splits;       /* 0 = registry choice, else 1, 2, 4 or 8: the most splits of a key
                             block's query range (blocks with a short range may get fewer) */
  int32_t lse_ld;         /* row length of lse and delta (>= GFA_LSE_LD(seq_len)) */
  int32_t stages;         /* 0 = all; else bitwise OR of GFA_BWD_DQ and GFA_BWD_DKV (profiling:
                             recomputing form: GFA_BWD_DKV alone reads the delta a previous
                             GFA_BWD_DQ wrote; materialised form: GFA_BWD_DKV runs delta and dK/dV,
                             GFA_BWD_DQ alone reads the dS store a previous GFA_BWD_DKV call left in
                             the same workspace) */
  void* workspace;        /* >= gfa_bwd_workspace_size(...) bytes when q_splits > 1; with
                             gfa_bwd_workspace_bytes(args) bytes the call runs the materialised
                             backward where that form exists */
  size_t workspace_bytes;
  void* stream;
  const int32_t* seg_lo;  /* the forward's segment table, or NULL */
  const int32_t* seg_hi;
  float softcap;          /* the forward's soft-cap (0 = off) */
  float dropout_p;        /* the forward's dropout probability and seed (0 = off) */
  uint64_t dropout_seed;
} gfa_bwd_args;

/* Tile configuration the library uses for one problem (mirrors the Python registry). */
typedef struct {
  int32_t head_dim;
  int32_t fwd_block_q;      /* query rows per forward workgroup */
  int32_t fwd_block_kv;     /* keys per LDS tile */
  int32_t fwd_waves;
  int32_t dq_block_q;
  int32_t dq_block_kv;
  int32_t dq_waves;
  int32_t dkv_block_kv;     /* keys per dKV workgroup */
  int32_t dkv_block_q;      /* queries per LDS tile */
  int32_t dkv_waves;
  int32_t q_splits;
} gfa_config_info;

/* Forward: O (and LSE unless lse == NULL). Returns a gfa_status. */
int gfa_fwd(const gfa_fwd_args* args);

/* Backward: delta, dQ, then dK/dV (summing Q-split fp32 partials when q_splits > 1).
 * Two forms, the same results to rounding:
 * - recomputing (the reference's, attention.py:1506-1620): the dQ kernel recomputes S, P and dP
 *   and computes delta in its prologue, then the dK/dV kernel;
 * - materialised: a delta kernel, the dK/dV kernel, which also stores every 32 x 32 block of dS
 *   it computes (16-bit, in the workspace), then dQ = scale * dS K from that store. It replaces
 *   two thirds of the dQ kernel's matrix work with 2 KiB of dS per block, written once and read
 *   once. Runs when the workspace holds the store (gfa_bwd_workspace_bytes), the store is within
 *   gfa_bwd_ds_limit and head_dim is 256 or 512 (soft-capping, dropout and segment tables
 *   included: the first two are in the stored dS, and the dQ kernel reads only the blocks the
 *   segment-trimmed dK/dV kernel writes); otherwise the recomputing form runs. */
int gfa_bwd(const gfa_bwd_args* args);

/* Bytes of the library-owned device scratch of gfa_bwd_noalloc, per GPU. */
#define GFA_NOALLOC_SCRATCH_BYTES (64u << 20)

/* gfa_bwd without caller-provided scratch. No counterpart in the reference: it is for callers
 * that cannot allocate device memory (code under HIP graph capture, tight serving or training
 * loops, harnesses that forbid hipMalloc). The caller passes inputs and outputs only: delta
 * and workspace must be NULL and workspace_bytes 0. delta and the Q-split partials live in a
 * file-scope device array of GFA_NOALLOC_SCRATCH_BYTES that each GPU the library runs on holds
 * until the process ends; the call itself allocates nothing. delta takes
 * batch * heads_q * lse_ld * 4 bytes (rounded up to 256) and the partials
 * gfa_bwd_workspace_size(...) bytes: a request beyond the scratch returns GFA_ERR_WORKSPACE.
 * q_splits = 0 takes the registry's split count, halved until its partials fit (1 needs none).
 * Every call on one GPU shares that GPU's scratch and leaves its contents there (a later
 * stages = GFA_BWD_DKV call reads the delta of the last GFA_BWD_DQ call): calls that overlap
 * on one GPU (concurrent streams or threads) race. It always runs the recomputing form (a dS
 * store does not fit a fixed scratch). Otherwise as gfa_bwd. */
int gfa_bwd_noalloc(const gfa_bwd_args* args);

/* Workspace bytes gfa_bwd needs for the given problem and q_splits (0 = registry choice) in the
 * recomputing form. */
size_t gfa_bwd_workspace_size(int32_t batch, int32_t heads_q, int32_t heads_kv, int32_t seq_len, int32_t head_dim,
                              int32_t causal, int32_t window, int32_t q_splits);

/* Workspace bytes of gfa_bwd(args) (the workspace fields are not read): the Q-split partials,
 * plus, where the materialised form applies, the dS store (batch * heads_q blocks of 2 KiB per
 * stored 32 x 32 (query tile, key tile) pair: per batch entry about heads_q * seq_len^2 bytes
 * under full causal masking, twice that without causal masking, 2 * heads_q * seq_len *
 * (window + 96) bytes with a sliding window). No counterpart in the reference. */
size_t gfa_bwd_workspace_bytes(const gfa_bwd_args* args);

/* Largest dS store the materialised backward uses, in bytes (default 32 GiB); a larger problem
 * runs the recomputing form, and 0 switches the materialised form off. A negative value only
 * queries. Process-wide; returns the limit before the call. No counterpart in the reference. */
int64_t gfa_bwd_ds_limit(int64_t bytes);

/* Fill *out with the configuration used for this problem without a sliding window (with a
 * window shorter than the sequence, the forward at head_dim 128 runs 32-key tiles, and the
 * dK/dV kernel at head_dim 256 runs role-split wave pairs, 64 keys per workgroup, two
 * workgroups per CU; gfa_bwd_workspace_size reports the split count for either; grids too small
 * to fill the GPU run 32-row workgroups in the forward and in dQ from the dS store). Returns a
 * gfa_status. */
int gfa_config(int32_t batch, int32_t heads_q, int32_t heads_kv, int32_t seq_len, int32_t head_dim,
               gfa_config_info* out);

/* Run-time work distribution of the long grids (no counterpart in the reference, whose grids the
 * Triton runtime launches as they are). With it on (the default), the forward and dQ kernels at
 * head_dim 512, when their grid exceeds one workgroup per CU, run as a persistent grid of one
 * workgroup per CU that takes the static grid's blocks, in their static order, from per-XCD
 * queues at run time (a faster XCD takes more blocks, no CU idles behind the hardware's in-order
 * dispatch). The queue counters live in a library-owned device array, one slot per launch out of
 * 256 used round-robin, zeroed by a one-workgroup kernel on the caller's stream before the
 * launch; the call still allocates nothing. Launches that overlap in time on different streams
 * must not share a slot: they must be fewer than 256 persistent launches apart. A launch captured
 * into a HIP graph keeps its slot for every replay, so graphs whose replays overlap on different
 * streams must not have been captured a multiple of 256 persistent launches apart (or must run
 * with this switched off). Every block computes exactly what it computes in the static grid, so
 * results are bit for bit the same either way. enable = 0 launches the static grids; a negative
 * value only queries. Process-wide; returns the setting before the call. */
int gfa_set_runtime_scheduling(int32_t enable);

/* Segment tables built on the device (no counterpart in the reference), each one launch on `stream`
 * that writes seg_lo and seg_hi, int32 (batch, seq_len) contiguous:
 * - from position ids, int32 or int64 (pos_bits 32 or 64), row b at pos + b * row_stride elements (0:
 *   one row for the whole batch): a sequence starts at token 0 and wherever the id is not the
 *   previous one plus one;
 * - from a padding mask, one byte per token (nonzero: a real token), row b at mask + b * row_stride:
 *   the row's real tokens are one segment. bad (int32, batch entries, device or host-mapped
 *   memory) receives 1 for a row whose real tokens are not one contiguous run, else 0; the table
 *   of such a row is not a partition.
 * seg_lo, seg_hi and bad must be 4-byte aligned, pos aligned to its type. Return a gfa_status. */
int gfa_segments_from_positions(const void* pos, int32_t pos_bits, int64_t row_stride, int32_t batch, int32_t seq_len,
                                int32_t* seg_lo, int32_t* seg_hi, void* stream);
int gfa_segments_from_mask(const uint8_t* mask, int64_t row_stride, int32_t batch, int32_t seq_len, int32_t* seg_lo,
                           int32_t* seg_hi, int32_t* bad, void* stream);

/* ---- Serving: a key/value cache held in 4 bits (no counterpart in the reference) ----
 *
 * A cache is two device arrays. `codes` (num_blocks, heads_kv, 2, block_size, head_dim / 2) bytes and
 * `scales` (num_blocks, heads_kv, 2, block_size, head_dim / 32) bytes hold blocks of block_size tokens
 * (a power of two, 32 to 1024) of K (side 0) and V (side 1). Format: MXFP4, 4.25 bits per
 * element: 32 neighbouring channels of a token and head share a power of two 2^e (its byte is
 * e + 127), an element is a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6. With amax the largest
 * magnitude of the 32, e = floor(log2 amax) - 2, one more where amax > 7 * 2^e, within [-125, 125] for
 * bf16 and [-23, 13] for fp16; elements round to the nearest value, ties to the even code, and
 * saturate at 6. A block that holds an infinity or a NaN has the byte 255 and reads as NaN; where it
 * is one of V, the token's first block of K has it too. The order of the bytes inside a head's block
 * is the kernels' own (csrc/gfa_kv4.h). `dtype` is the type of the rows written, read and
 * attended with.
 *
 * A token's place is its slot, block * block_size + offset. A request's blocks stand in its row of a
 * block table, position p of it in block table[p / block_size]; entries outside [0, num_blocks) are
 * no block. Token rows are (batch, heads, seq_len, head_dim) tensors with a unit-stride head dim, 16-byte
 * aligned rows and strides that are multiples of 8 elements; token t of a call is row t % seq_len of
 * batch entry t / seq_len (a packed step has batch 1, a step of single tokens may have seq_len 1). */
typedef struct {
  void* codes;
  void* scales;
  int32_t num_blocks, heads_kv, block_size, head_dim;
  int32_t dtype; /* gfa_dtype */
} gfa_kv4_cache;

/* Rows to the cache (gfa_kv4_write: k and v are read) or from it (gfa_kv4_read: k and v are written). */
typedef struct {
  gfa_kv4_cache cache;
  void* k; /* (batch, heads_kv, seq_len, head_dim) */
  void* v;
  gfa_strides k_strides, v_strides;
  int32_t batch, seq_len;
  const int64_t* slots; /* (batch * seq_len); outside [0, num_blocks * block_size): writes nothing, reads zeros.
                           Slots of one write must differ: a slot given twice ends with bytes of both rows. */
  void* stream;
} gfa_kv4_rows_args;

int gfa_kv4_write(const gfa_kv4_rows_args* args);
int gfa_kv4_read(const gfa_kv4_rows_args* args);

/* A step's plan: request b holds lens[b] tokens and gets fresh[b] more (negative counts are 0), packed
 * in the order of the requests. It holds ceil(lens / block_size) blocks; further ones it needs are the
 * next entries of free_ids behind the *used that are taken, handed out in the order of the requests
 * and entered in its row of the table. Where the free list ends, -1 is entered: *used_out above
 * free_count tells of it. Blocks past the table's width are handed out too, and entered nowhere. One launch; the inputs other
 * than the table are only read, the outputs must not overlap them. */
typedef struct {
  const int32_t* lens;  /* (requests) */
  const int32_t* fresh; /* (requests) */
  int32_t* table;       /* (requests, table_width), rows table_stride apart */
  int64_t table_stride;
  const int32_t* free_ids; /* (free_count) */
  const int32_t* used;     /* (1) */
  int32_t requests, table_width, free_count, block_size;
  int32_t tokens;     /* length of slots and positions */
  int64_t* slots;     /* (tokens): the new tokens' slots; -1 where there is no block, behind the last token or
                         past the table's width */
  int32_t* positions; /* (tokens): their positions in their requests (0 behind the last) */
  int32_t* cu;        /* (requests + 1): first token of each request, at most `tokens` */
  int32_t* lens_out;  /* (requests): lens + fresh */
  int32_t* used_out;  /* (1) */
  void* stream;
} gfa_kv4_plan_args;

int gfa_kv4_plan(const gfa_kv4_plan_args* args);

/* Attention of a step's new tokens over the cache, the new tokens' own keys and values in it. Request b has
 * lens[b] tokens altogether, its new ones are the last cu[b + 1] - cu[b] of them and stand in q from
 * token cu[b] on (cu NULL: every request has batch * seq_len / requests). New token i, at position
 * p = lens - fresh + i, attends to positions <= p, with a window W > 0 only to those > p - W; without
 * causal to all lens positions. Positions without a block are not attended to; a row that attends to
 * nothing is zero, and so are rows of no request (ahead of cu[0], from cu[requests] on). max_new, when not
 * 0, is the most new tokens of any request and only chooses the kernel. Values in the tables, lens and cu cannot make the call
 * address memory outside its arrays. */
typedef struct {
  gfa_kv4_cache cache;
  const void* q; /* (batch, heads_q, seq_len, head_dim) */
  void* o;
  gfa_strides q_strides, o_strides;
  int32_t batch, heads_q, seq_len, requests;
  const int32_t* table; /* (requests, table_width), rows table_stride apart */
  int64_t table_stride;
  const int32_t* lens; /* (requests) */
  const int32_t* cu;   /* (requests + 1) or NULL */
  int32_t table_width, causal, window, max_new;
  float scale, softcap; /* softcap 0 = off */
  void* workspace;      /* >= gfa_kv4_attn_workspace_bytes(args), 16-byte aligned */
  size_t workspace_bytes;
  void* stream;
  /* gfa_kv4_share's results for this table, lens and cu, or NULL: the groups' prefixes are attended to once for all of a
   * group's queries, where their lengths promise that it is faster (shared_apart 0) or wherever there is a group (1). Tables too narrow
   * to gain by it take the call without; in wide ones a call that finds little in common can take some us longer. The same
   * result within the same bound: weights are rounded against other maxima, and 32-bit sums taken in another order. Without
   * effect with a window and where max_new (0: the average) times heads_q / heads_kv are many; with max_new 0 single requests of
   * many rows are computed as without. */
  const int32_t* shared_skip; /* (requests) */
  const int32_t* shared_cu;   /* (requests + 1) */
  const int32_t* shared_lens; /* (requests) */
  int32_t shared_apart;
} gfa_kv4_attn_args;

int gfa_kv4_attn(const gfa_kv4_attn_args* args);
/* Workspace of gfa_kv4_attn(args) in bytes; pointers are not read, but for whether cu is NULL. */
size_t gfa_kv4_attn_workspace_bytes(const gfa_kv4_attn_args* args);

/* ---- Requests with something in common ----
 *
 * Pages. Rows of a block table may hold the same blocks. caches is a host array of the layers' caches, all of one num_blocks (at
 * most 2^18) and block_size, whose blocks the table's rows hold; at most 4096 requests and rows. Entries of the table outside
 * [0, num_blocks) are no block, request b holds the first ceil(lens[b] / block_size). Values in the arrays cannot
 * make a call address memory outside them.
 *
 * gfa_kv4_fork: the block tables of the next step's requests. Row r takes request parents[r] (outside [0, requests): an empty
 * row; NULL: request r) and keeps its first min(lens, keep[r]) tokens (keep NULL: all). A block of which a row keeps only a part is
 * the row's to write to: it stays with the first such row if no row keeps it whole, and every other such row gets a copy
 * of it, in every cache. Blocks of the requests that no row holds any more are given back: in ascending order they become the
 * last ones ahead of *used in free_ids (at most *used of them). Copies take, in the order of the rows, the blocks just given
 * back and then the entries from *used on; where the list ends the row's entry is -1, and *used_out above free_count tells of it.
 * gfa_kv4_compact: of the n blocks that requests hold, the k-th (in ascending order) at or past n is moved, in every cache, to
 * the k-th block below n that no request holds; free_ids (num_blocks entries: all of the pool) becomes 0, 1, ... and *used_out n.
 * parents, keep, rows, used and lens_out are not read.
 * table_out (rows, compact: requests; table_width) and lens_out must not overlap the inputs. Two launches and more: the tables
 * first, then the blocks' bytes. */
typedef struct {
  const gfa_kv4_cache* caches;
  int32_t layers;
  const int32_t* table; /* (requests, table_width), rows table_stride apart */
  int64_t table_stride;
  const int32_t* lens; /* (requests) */
  int32_t requests, table_width;
  const int32_t* parents; /* (rows) or NULL */
  const int32_t* keep;    /* (rows) or NULL */
  int32_t rows;
  int32_t free_count;
  int32_t* free_ids;   /* (free_count), changed in place */
  const int32_t* used; /* (1) */
  int32_t* table_out;  /* (rows, table_width) */
  int32_t* lens_out;   /* (rows) */
  int32_t* used_out;   /* (1) */
  void* workspace;     /* >= gfa_kv4_pages_workspace_bytes, 4-byte aligned */
  size_t workspace_bytes;
  void* stream;
} gfa_kv4_pages_args;

int gfa_kv4_fork(const gfa_kv4_pages_args* args);
int gfa_kv4_compact(const gfa_kv4_pages_args* args);
/* Workspace of gfa_kv4_fork with so many rows, or of gfa_kv4_compact of so many blocks. */
size_t gfa_kv4_pages_workspace_bytes(int32_t rows_or_blocks);

/* Copies block src[i] to block dst[i] in every cache; pairs with an id outside [0, num_blocks) are left out. No block may be a
 * destination twice, or a destination and a source. */
int gfa_kv4_copy(const gfa_kv4_cache* caches, int32_t layers, const int32_t* src, const int32_t* dst, int32_t pairs, void* stream);

/* What neighbouring requests of a step have in common, as gfa_kv4_attn takes it: the whole blocks that a request's row and the row
 * before it begin with, ahead of both requests' new tokens (cu). Neighbours with at least `least` tokens in common are a group, the
 * fewest tokens that two neighbours in it have in common are its prefix. skip (requests): tokens of the request's prefix, 0
 * without a group; cu_out (requests + 1) and lens_out (requests): the groups' new tokens as one request's, cu_out[b + 1] -
 * cu_out[b] of them over lens_out[b] tokens (0 for all requests but a group's first). At most 4096 requests. */
typedef struct {
  const int32_t* table; /* (requests, table_width), rows table_stride apart */
  int64_t table_stride;
  const int32_t* lens; /* (requests): tokens with the new ones */
  const int32_t* cu;   /* (requests + 1) */
  int32_t requests, table_width, block_size, least;
  int32_t* skip;
  int32_t* cu_out;
  int32_t* lens_out;
  void* stream;
} gfa_kv4_share_args;

int gfa_kv4_share(const gfa_kv4_share_args* args);

/* Verification of drafted tokens. Request b's tokens of the step are cu[b] .. cu[b + 1] - 1 (cu NULL: token_count / requests
 * each): its last known token and the drafted ones. target (token_count, vocab): row t the target's probabilities of what follows
 * token t; draft: row t the probabilities that token t was drawn from (not read for a request's first; NULL: the tokens were
 * proposed for certain). Token t is accepted, in the order of a request's, while accept[t] * draft[t, x] < target[t - 1, x], x = tokens[t]
 * (a token outside the vocabulary is not). Behind the accepted ones a token is drawn: where one was not accepted from max(target -
 * draft, 0), else from the target: the first entry at which the running sum of weights exceeds sample[b] times their sum, in 64 bits.
 * Where no weight is left the target's probabilities are taken instead, and without any of those the token is -1. What is
 * not a finite positive number counts as probability 0, sample as the nearest in [0, 1].
 * follows[t]: the token that follows token t in the request: a drafted one that was accepted, the drawn one, then -1 (also for
 * tokens of no request). accepted (requests): drafted tokens accepted. lens_out = lens less the drafted tokens that were not. */
typedef struct {
  const void* target;
  const void* draft;
  int64_t target_stride, draft_stride; /* elements from row to row */
  int32_t type;                        /* 0 fp16, 1 bf16, 2 fp32 */
  int32_t token_count, vocab, requests;
  const int64_t* tokens; /* (token_count) */
  const float* accept;   /* (token_count), uniform in [0, 1) */
  const float* sample;   /* (requests), uniform in [0, 1) */
  const int32_t* lens;   /* (requests) */
  const int32_t* cu;     /* (requests + 1) or NULL */
  int64_t* follows;      /* (token_count) */
  int32_t* accepted;     /* (requests) */
  int32_t* lens_out;     /* (requests) */
  void* workspace;       /* >= gfa_kv4_verify_workspace_bytes(requests, vocab), 8-byte aligned */
  size_t workspace_bytes;
  void* stream;
} gfa_kv4_verify_args;

int gfa_kv4_verify(const gfa_kv4_verify_args* args);
size_t gfa_kv4_verify_workspace_bytes(int32_t requests, int32_t vocab);

/* Message of the last failing call on this thread ("" if none). */
const char* gfa_last_error(void);

/* GFA_VERSION of the built library. */
int gfa_version(void);

#ifdef __cplusplus
}
#endif

#endif /* GFA_H_ */
