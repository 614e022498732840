/*
 * q4rdna.h -- C ABI of the MI355X (gfx950) Q4_RDNA group-64 dequant-GEMV.
 *
 * A drop-in for the reference's llama.cpp entry points
 * (source/q4rdna.cuh:5-24, defined at source/q4rdna.cu:713-793) with ggml
 * types replaced by plain pointers and sizes.  The packed layout is the
 * reference's byte-exact Q4_RDNA sidecar: 32-row tiles of 1088 bytes (32 fp16
 * scales, then 32x32 lane-interleaved bytes of two's-complement nibbles, low
 * nibble = even k) in (row tile, group) order.
 *
 * Conventions
 *  - Every call returns a status.  Q4RDNA_NOT_APPLICABLE is the reference's
 *    "return false": the call touched nothing and the caller should run its
 *    own path.  Negative values are errors; q4rdna_last_error() describes the
 *    last one on the calling thread.
 *  - Device pointers are caller-owned except the sidecar's weights, which the
 *    library owns until q4rdna_sidecar_close().
 *  - `stream` is a hipStream_t (NULL = the null stream).  Launches are
 *    asynchronous on that stream; nothing here synchronises it.
 *  - A launch needs the weights' device to be the current device.
 */
#ifndef Q4RDNA_H
#define Q4RDNA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define Q4RDNA_ABI_VERSION 4

/* status codes */
#define Q4RDNA_OK 0
#define Q4RDNA_NOT_APPLICABLE 1
#define Q4RDNA_ERR_ARGUMENT (-1)
#define Q4RDNA_ERR_FORMAT (-2)
#define Q4RDNA_ERR_IO (-3)
#define Q4RDNA_ERR_HIP (-4)
#define Q4RDNA_ERR_MEMORY (-5)

/* format constants (source/q4rdna.cu:20-22) */
#define Q4RDNA_GROUP 64
#define Q4RDNA_TILE_ROWS 32
#define Q4RDNA_TILE_BYTES 1088

/* scale-search algorithms of the packers */
#define Q4RDNA_ALGO_SIDECAR 0 /* source/q4rdna_sidecar_pack.cpp:126-179 */
#define Q4RDNA_ALGO_ABSMAX 1  /* source/q4rdna_cpu_experiment.cpp:209-211 */
#define Q4RDNA_ALGO_RANGE 2   /* source/q4rdna_cpu_experiment.cpp:213-223 */
#define Q4RDNA_ALGO_MSE 3     /* source/q4rdna_cpu_experiment.cpp:225-236 */

/* GLU operations accepted by q4rdna_mul_mat_glu (source/q4rdna.cu:776) */
#define Q4RDNA_GLU_SWIGLU 0

/* A packed tensor resident on a device: rows x columns weights, rows%32 == 0,
 * columns%64 == 0, `tiles` 16-byte aligned, rows*columns*34/64 bytes. */
typedef struct q4rdna_weight {
    const uint8_t *tiles;
    uint32_t rows;
    uint32_t columns;
    int32_t device;
    uint32_t reserved;
} q4rdna_weight;

typedef struct q4rdna_sidecar q4rdna_sidecar;

/* Library version (Q4RDNA_ABI_VERSION) and the last error on this thread. */
int q4rdna_abi_version(void);
const char *q4rdna_last_error(void);

/* ---- sidecar container --------------------------------------------------
 * q4rdna_sidecar_inspect: host-only validation of a sidecar image prefix that
 * holds at least the header and the index; `file_size` is the size of the
 * whole file.  Applies the loader's acceptance rules of
 * source/q4rdna.cu:129-155 (magic, version, group 64, 32 rows, 1088-byte
 * tiles, NUL-terminated names, offsets inside the data region, rows%32,
 * columns%64, size = rows*columns*34/64) and the data-length check of
 * source/q4rdna.cu:163-170.  On success *count receives the entry count. */
int q4rdna_sidecar_inspect(const void *image, uint64_t image_size, uint64_t file_size,
                           uint32_t *count);

/* Open a sidecar file and upload its data region to `device` once
 * (source/q4rdna.cu:119-179, without the device-0 restriction). */
int q4rdna_sidecar_open(const char *path, int device, q4rdna_sidecar **out);
/* Same from an in-memory image of `size` bytes. */
int q4rdna_sidecar_open_memory(const void *image, uint64_t size, int device, q4rdna_sidecar **out);
/* Frees the sidecar's device buffer (hipFree waits for work in flight):
 * every q4rdna_weight found in it is invalid afterwards.  Not for the
 * process-wide sidecar of q4rdna_default_sidecar, which lives until exit. */
void q4rdna_sidecar_close(q4rdna_sidecar *sidecar);
uint32_t q4rdna_sidecar_count(const q4rdna_sidecar *sidecar);
/* Entry metadata; name receives up to 64 bytes including the NUL. */
int q4rdna_sidecar_entry(const q4rdna_sidecar *sidecar, uint32_t index, char name[64],
                         uint32_t *rows, uint32_t *columns, uint64_t *offset, uint64_t *size);

/* Name lookup with the reference's shape check: `ne0` = columns (K) and
 * `ne1` = rows (M) as ggml stores them.  NOT_APPLICABLE when the name is
 * absent or the shape differs (source/q4rdna.cu:682-705). */
int q4rdna_find(const q4rdna_sidecar *sidecar, const char *name, int64_t ne0, int64_t ne1,
                q4rdna_weight *out);

/* Describe tiles already resident on `device` (synthetic or externally
 * uploaded tensors). */
int q4rdna_weight_from_device(const void *tiles, uint32_t rows, uint32_t columns, int device,
                              q4rdna_weight *out);

/* Sidecar named by LLAMA_Q4_RDNA_SIDECAR, opened once per process on the
 * first call (source/q4rdna.cu:683,698) on that call's device, and kept
 * until exit (never pass it to q4rdna_sidecar_close).  NULL when unset or
 * invalid, or for another device. */
q4rdna_sidecar *q4rdna_default_sidecar(int device);
/* The reference's LLAMA_Q4_RDNA_SCOPE name filter (source/q4rdna.cu:685-696):
 * scope NULL/"" admits every name; "ffn", "qkv-fallback", "hotspot", "attn"
 * as in the reference.  Returns 1 if `name` is in scope, else 0. */
int q4rdna_scope_allows(const char *scope, const char *name);

/* ---- GEMV entry points ---------------------------------------------------
 * y[M] = W[M][K] x[K] in fp32 accumulation.  x_ne0 must equal K and y_ne0 M
 * (the reference's src1->ne[0] / dst->ne[0] checks); any mismatch, a weight
 * on another device or a NULL weight returns NOT_APPLICABLE with nothing
 * launched.  x and y are contiguous fp32 device buffers (4-byte aligned);
 * y may not overlap x, and an add vector is either y itself or apart from
 * it (argument errors otherwise).
 *
 * Launches with split K use a scratch buffer per (device, stream).  The
 * first call that needs more than the stream has allocates it, which it
 * cannot do while that stream is being captured (other streams may be): make
 * one call of each shape on the stream before capturing.  (A policy-chosen
 * split of a tall matrix or group, captured without that call, takes fewer
 * chunks instead, so another order of each row's sum and other last bits than
 * the eager call's; it is refused only where these need a larger buffer too.)
 * Outgrown buffers are never freed, so a graph captured earlier stays
 * valid.  Calls on one stream are ordered by it; a graph must not replay on
 * another stream while the stream it was captured on runs such calls.
 *
 * Replaces ggml_cuda_q4rdna_mul_mat (source/q4rdna.cuh:5-9, q4rdna.cu:713-745). */
int q4rdna_mul_mat(const q4rdna_weight *w, const float *x, int64_t x_ne0, float *y, int64_t y_ne0,
                   void *stream);

/* y = W x + add, add[M] fp32.
 * Replaces ggml_cuda_q4rdna_mul_mat_add (source/q4rdna.cuh:11-16, q4rdna.cu:747-767). */
int q4rdna_mul_mat_add(const q4rdna_weight *w, const float *x, int64_t x_ne0, const float *add,
                       int64_t add_ne, float *y, int64_t y_ne0, void *stream);

/* y = (W_up x) * silu(W_gate x), both weights of one shape; glu_op must be
 * Q4RDNA_GLU_SWIGLU (anything else is NOT_APPLICABLE).
 * Replaces ggml_cuda_q4rdna_mul_mat_glu (source/q4rdna.cuh:18-24, q4rdna.cu:769-793). */
int q4rdna_mul_mat_glu(const q4rdna_weight *up, const q4rdna_weight *gate, const float *x,
                       int64_t x_ne0, int glu_op, float *y, int64_t y_ne0, void *stream);

/* Launch options: split_k = number of K chunks reduced across workgroups of
 * the per-tensor kernel (0 = the shape policy, the reference's launch policy
 * at source/q4rdna.cu:578-680 and its LLAMA_Q4_RDNA_COOP override
 * :579-584); kernel = Q4RDNA_KERNEL_POLICY or Q4RDNA_KERNEL_VALU (the same
 * kernel) or Q4RDNA_KERNEL_SEQUENTIAL (any other value, 2 included, which
 * ABI 1 used for a kernel since withdrawn, is an argument error); reserved
 * words must be zero.  Zero-initialised options mean "policy" throughout. */
#define Q4RDNA_KERNEL_POLICY 0
#define Q4RDNA_KERNEL_VALU 1 /* the split-K VALU kernel (split_k applies) */
/* The reference's old mapping (LLAMA_Q4_RDNA_MAPPING=old, source/q4rdna.cu:
 * 190-234,626-634): one thread per row, its weights in k order, one fp32 fma
 * each, so y is bit for bit the reference bench's CPU loop
 * (source/q4rdna_gemv_bench.hip:189-210) before the epilogue.  split_k must be 0
 * or 1; q4rdna_mul_mat_batch runs it once per vector, q4rdna_mul_mat_group
 * refuses it (argument error).  Slow: an ablation and a bit-exact
 * reference, not a decode path. */
#define Q4RDNA_KERNEL_SEQUENTIAL 3
typedef struct q4rdna_launch_options {
    uint32_t split_k;
    uint32_t kernel;
    uint32_t reserved[6];
} q4rdna_launch_options;

/* q4rdna_mul_mat / _add / _glu with explicit options (add, gate may be NULL). */
int q4rdna_mul_mat_ex(const q4rdna_weight *w, const q4rdna_weight *gate, const float *x,
                      const float *add, float *y, const q4rdna_launch_options *options,
                      void *stream);

/* n = 1..Q4RDNA_MAX_BATCH activation vectors against one weight in one
 * launch (no reference counterpart: the reference's hooks decline batches
 * above 1, source/q4rdna.cu:722,754,777).  x holds n vectors of `columns`
 * floats back to back, y (and add) n rows of `rows` floats, as ggml's src1
 * and dst with ne[1] = n, contiguous.  gate (may be NULL) makes it the
 * SwiGLU site.  options->split_k as in q4rdna_mul_mat_ex (0 = the shape
 * policy, for n >= 2 with its own choice for tall and uneven shapes); for
 * n >= 2 it is raised until every K chunk holds at most 32 groups (16 for
 * n > 4).  Each tile is read once for all n vectors; each
 * vector's result is bit-identical to q4rdna_mul_mat_ex of that vector with
 * that split where that call runs eight-wave workgroups. */
int q4rdna_mul_mat_batch(const q4rdna_weight *w, const q4rdna_weight *gate, const float *x, uint32_t n,
                         const float *add, float *y, const q4rdna_launch_options *options,
                         void *stream);

/* Several GEMVs that share one activation, in one launch: y_i = W_i x
 * (+ add_i), or with gate_tiles y_i = (W_i x + add_i) * silu(G_i x) -- e.g.
 * q, k and v of a decoder layer, or its gate and up projections.  count =
 * 1..Q4RDNA_MAX_GROUP; every weight has K = x_ne0 columns (else
 * NOT_APPLICABLE) and lives on the current device; gate_tiles is given for
 * every descriptor or for none, each of its weight's shape; no y may overlap
 * x, another descriptor's y or another descriptor's add, and a descriptor's
 * add is its own y or apart from it (argument error).  x is read once per
 * workgroup in the kernel (no separate prepare launch).  options->split_k
 * applies (0 = the shape policy for the group's total rows, raised until
 * every K chunk holds at most 64 groups; K above 262,144 columns, 64 chunks
 * of 64 groups, is NOT_APPLICABLE).  Each output equals q4rdna_mul_mat_ex of
 * its weight at the group's split bit for bit when both launches run the
 * same workgroup width: eight waves, which each launch uses while it has at
 * most four workgroups per CU (rows / 32 * split of the whole group, or of
 * the one weight), and four waves above that.  The split-K scratch is the stream's,
 * as for q4rdna_mul_mat.  No reference counterpart: the reference launches
 * one kernel per projection and fuses only gate/up
 * (source/q4rdna.cu:736-741,769-793). */
#define Q4RDNA_MAX_GROUP 8
typedef struct q4rdna_group_desc {
    q4rdna_weight weight;      /* W (the up projection for SwiGLU) */
    const uint8_t *gate_tiles; /* SwiGLU gate tiles of W's shape, or NULL */
    const float *add;          /* [rows] or NULL */
    float *y;                  /* [rows] */
} q4rdna_group_desc;
int q4rdna_mul_mat_group(const q4rdna_group_desc *descs, uint32_t count, const float *x, int64_t x_ne0,
                         const q4rdna_launch_options *options, void *stream);

/* Split-K factor the shape policy picks for rows x columns on `device`,
 * without a SwiGLU gate (single launches with one may take more chunks). */
uint32_t q4rdna_policy_split_k(uint32_t rows, uint32_t columns, int device);

/* q4rdna_mul_mat_ex that allocates nothing.  No counterpart in the
 * reference: it is for callers that cannot allocate (code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc).  The K
 * chunks of a split launch meet in exchange slots, which here live in a
 * fixed per-GPU device array of Q4RDNA_NOALLOC_SLOTS 32-bit slots (8 MiB,
 * held by every GPU the library runs on until the process ends).  A launch
 * at split_k s > 1 needs (p - 1) * rows slots, p the smallest power of two
 * >= s, doubled with a gate; one that would need more returns
 * Q4RDNA_ERR_ARGUMENT and launches nothing.  Arguments, statuses and results
 * are those of q4rdna_mul_mat_ex (bit-identical at the same split).  Every
 * call on a GPU shares that GPU's array: calls that overlap on one GPU race,
 * so issue them on one stream or order them with events.  The first call on
 * a GPU looks the array's address up; its slots are zero from the start (a
 * zero-initialised device variable, left zero by every launch), so no set-up
 * runs on any stream and the first call may be captured into a graph. */
#define Q4RDNA_NOALLOC_SLOTS (1u << 21)
int q4rdna_mul_mat_ex_noalloc(const q4rdna_weight *w, const q4rdna_weight *gate, const float *x,
                              const float *add, float *y, const q4rdna_launch_options *options,
                              void *stream);

/* ---- multi-tensor stack --------------------------------------------------
 * One launch that sweeps many independent GEMVs (a decode step's weight
 * streaming).  The GEMVs run concurrently and in an order the plan picks
 * (longest K chunks first), so no descriptor's x, add or y may overlap
 * another's y, and an add is its own y or apart from it (plan creation
 * refuses these with an argument error).  A descriptor's x may overlap its
 * own y: the prepare launch reads every x before the sweep writes.  No
 * reference counterpart: the reference launches one kernel per tensor
 * (source/q4rdna.cu:736-741). */
typedef struct q4rdna_gemv_desc {
    q4rdna_weight weight;      /* W (the up projection for SwiGLU) */
    const uint8_t *gate_tiles; /* SwiGLU gate tiles of the same shape, or NULL */
    const float *x;            /* [columns], 16-byte aligned */
    const float *add;          /* [rows] or NULL */
    float *y;                  /* [rows] */
} q4rdna_gemv_desc;

typedef struct q4rdna_plan q4rdna_plan;

/* Build a plan for `count` descriptors (uploads the descriptor table once).
 * Plans also fix here which workgroup runs which item: a load-balancing deal
 * computed on the host, about 2 ms for the 252-tensor Qwen3-8B stack and
 * 0.2 s for 100,000 items. */
int q4rdna_plan_create(const q4rdna_gemv_desc *descs, uint32_t count, int device,
                       q4rdna_plan **out);
/* Batched plan: every descriptor's x holds n activation vectors of
 * `columns` floats one after another ([n][columns]), y and add hold n
 * results of `rows` floats ([n][rows]); n = 1..Q4RDNA_MAX_BATCH (the
 * small-batch decode shapes).  A plan with little work per workgroup cuts
 * long rows into more K chunks, so the order of a row's sum, and with it the
 * last bits, depends on the shapes in the plan (not on n, the values or the
 * order of the descriptors; a single-vector plan's sums depend on their own
 * shape alone).  No reference counterpart: the reference's hooks decline
 * batches above 1 (source/q4rdna.cu:722,754,777). */
#define Q4RDNA_MAX_BATCH 8
int q4rdna_plan_create_batch(const q4rdna_gemv_desc *descs, uint32_t count, uint32_t n, int device,
                             q4rdna_plan **out);
/* Launch the whole plan on `stream` (prepare + sweep); allocates nothing.
 * Launches of one plan share its digit buffers, split-K partials and
 * counters, so they must not overlap: keep them on one stream or order
 * them with events.  Different plans are independent. */
int q4rdna_plan_launch(q4rdna_plan *plan, void *stream);
/* The two launches of q4rdna_plan_launch, for callers that time or overlap
 * them: prepare converts every activation x into the plan's int8 digit
 * buffers; sweep runs the GEMVs and must follow a prepare of the same x on
 * the same stream. */
int q4rdna_plan_prepare(q4rdna_plan *plan, void *stream);
int q4rdna_plan_sweep(q4rdna_plan *plan, void *stream);
void q4rdna_plan_destroy(q4rdna_plan *plan);
/* Workgroups the plan launches (persistent grid). */
uint32_t q4rdna_plan_workgroups(const q4rdna_plan *plan);

/* Launch statistics, the reference's q4rdna_launches and per-entry hits
 * (source/q4rdna.cu:57,73,706-709,742,764,789-791).  Every GEMV kernel
 * launch the entry points above make counts once (q4rdna_mul_mat_batch's
 * per-vector launches one each, a plan's sweep once), and every weight it
 * streams that starts an entry of an open sidecar counts a hit for that
 * entry (a SwiGLU launch hits both weights). */
uint64_t q4rdna_launch_count(void);
/* Hits of entry `index` of `sidecar` (0 for an invalid pair). */
uint64_t q4rdna_sidecar_hits(const q4rdna_sidecar *sidecar, uint32_t index);
/* The reference's report on stderr (source/q4rdna.cu:75-112, same lines):
 * "Q4_RDNA: launched N decode GEMV kernels", with LLAMA_Q4_RDNA_TRACE set
 * one "Q4_RDNA: hit <name> <hits>" line per entry that was hit, and the
 * unique / hits-by-shape summary, over every open sidecar.  Printed at
 * process exit once q4rdna_default_sidecar has loaded (source/q4rdna.cu:176). */
void q4rdna_report_stats(void);

/* ---- packing and dequantisation ------------------------------------------
 * Quantize fp32 W[rows][columns] (device, row-major) into tiles (device) with
 * the chosen scale search, bit-identical to the reference CPU packers
 * (source/q4rdna_sidecar_pack.cpp:126-179,259-279 for Q4RDNA_ALGO_SIDECAR;
 * source/q4rdna_cpu_experiment.cpp:136-273,387-399 for absmax/range/mse). */
int q4rdna_pack(const float *w, uint32_t rows, uint32_t columns, int algorithm, uint8_t *tiles,
                void *stream);

/* Test/inspection: out[rows][columns] = fp32(scale) * code, the exact
 * product (source/q4rdna_cpu_experiment.cpp:270-271). */
int q4rdna_dequantize(const q4rdna_weight *w, float *out, void *stream);

/* ---- the rest of a decoder layer -------------------------------------------
 * What a program runs between the GEMVs above: cache append, attention and
 * norm.  No reference counterpart (its llama.cpp host runs these).  The
 * launches are asynchronous on `stream`; activations are fp32, fp16 or bf16
 * and every sum, softmax statistic and norm is kept in fp32. */
#define Q4RDNA_F32 0
#define Q4RDNA_F16 1
#define Q4RDNA_BF16 2

/* A paged key/value cache of one layer, in caller-owned device buffers.
 * Pages are blocks of Q4RDNA_KV_BLOCK tokens.  A full block holds int8 codes
 * with one fp32 scale per head for K and one for V (x = code * scale).  The
 * last, partly filled block of a sequence is held in the sequence's slot with
 * 16-bit codes, as two int8 planes (256 * high + low, |code| <= 32512), and an
 * fp32 scale per token and head (absmax / 32512).  When a block fills, its
 * scale becomes 256 * the largest of its tokens' scales and each code
 * rint(code16 * (token scale / scale)), in fp32: every number is rounded to 16 bits
 * once and to 8 bits once, so the cache's bytes do not depend on the chunks in
 * which the tokens arrive, and a full page never changes again (sequences may
 * share it).  A slot holds two blocks, used in turn: those of the greatest
 * length m that the sequence has had and of the block before.  So tokens may be
 * taken back to any length >= 64 * (m / 64 - 1), the last full block included,
 * and the sequence be appended to from there, as long as no other one reads
 * that page; cut back to length 0, or in a new slot, it starts afresh.
 *
 * The order of codes within a block of one head, 16 bytes per lane of a
 * 64-lane int8 matrix instruction:
 *   K  token 16 n + c, number 64 s + 16 g + j at (((n * D/64 + s) * 4 + g) * 16 + c) * 16 + j
 *   V  token 16 a + 4 g + b, number 16 n + c  at ((n * 4 + g) * 16 + c) * 16 + 4 a + b
 * A token with a number that is not finite has the scale NaN and reads as NaN,
 * and so does its block once full; one whose largest number is under 1e-30
 * reads as zero. */
#define Q4RDNA_KV_BLOCK 64
typedef struct q4rdna_kv_cache {
    int8_t *pages;        /* [page_count][kv_heads][2 (K, V)][64 * head_dim], 16-byte aligned */
    float *scales;        /* [page_count][kv_heads][2], 8-byte aligned */
    int8_t *open;         /* [slot_count][2][kv_heads][4 (K high, K low, V high, V low)][64 * head_dim], 16-byte aligned */
    float *open_scales;   /* [slot_count][2][kv_heads][2 (K, V)][64], 16-byte aligned */
    uint32_t *faults;     /* counts what the kernels refused (see q4rdna_kv_batch), or NULL */
    uint32_t page_count;
    uint32_t slot_count;
    uint32_t kv_heads;
    uint32_t head_dim;    /* 64 or 128 */
    int32_t device;       /* of the buffers: the calls run there, whatever the current device is */
    uint32_t reserved;
} q4rdna_kv_cache;

/* The sequences of one step, shared by the calls of all layers.  The arrays
 * are device memory and are read when the kernels run, so a captured graph
 * may be replayed with other lengths, tables and slots in them.  Sequence i
 * has `past[i]` tokens in the cache before the step and the step's tokens
 * cu_tokens[i] .. cu_tokens[i + 1] - 1 (cu_tokens NULL: one token each,
 * tokens == sequences) at the positions past[i], past[i] + 1, ...  Its token t
 * lies in page table[i * table_width + t / 64].  slots[i] is its slot (NULL:
 * slot i).  max_tokens bounds every sequence's tokens in the step.
 * The kernels check what they read: a sequence whose entries are out of range
 * (tokens outside the step's or more than max_tokens, past < 0, past + tokens
 * > 64 * table_width, a bad slot) is skipped, its results not written; a page
 * outside the cache is not written, and rows that need to read it come out as
 * NaN.  Each adds to *faults.
 * A call is made before the lengths are known: table_width bounds them, and a
 * table no wider than the sequences may become is the faster one. */
typedef struct q4rdna_kv_batch {
    const int32_t *past;      /* [sequences] */
    const int32_t *cu_tokens; /* [sequences + 1], ascending, or NULL */
    const int32_t *table;     /* [sequences][table_width] */
    const int32_t *slots;     /* [sequences] or NULL */
    uint32_t sequences;       /* at most 65535 */
    uint32_t tokens;          /* of all sequences in this step */
    uint32_t max_tokens;
    uint32_t table_width;     /* at most 2^24 */
} q4rdna_kv_batch;

/* Rows of activations [tokens][heads][head_dim]: the numbers of a head are
 * contiguous, the strides are in elements. */
typedef struct q4rdna_kv_rows {
    void *data;
    int64_t token_stride;
    int64_t head_stride;
} q4rdna_kv_rows;

/* Append the step's keys and values.  Each head's row of q and k is first
 * normalised (x * rsqrt(mean x^2 + eps) * weight) where q_norm / k_norm is
 * given, then its first `rotary` numbers are rotated by the token's position
 * p: pairs (x_i, x_{i + rotary/2}), or (x_{2i}, x_{2i+1}) with `interleaved`,
 * become (a cos - b sin, b cos + a sin) with cos[p][i], sin[p][i].  Rotated q
 * goes to q_out (which may be q); rotated k and v go into the cache.
 * rotary is a multiple of 8 up to head_dim, 0 for no rotation; a sequence that
 * reaches past the `positions` rows of cos and sin is skipped as above. */
typedef struct q4rdna_kv_append_desc {
    uint32_t dtype;           /* of k, v, q and q_out */
    uint32_t q_heads;         /* a multiple of kv_heads; 0: no q */
    q4rdna_kv_rows k, v, q, q_out;
    const float *cos, *sin;   /* [positions][rotary / 2], 16-byte aligned */
    uint32_t positions;
    uint32_t rotary;
    uint32_t interleaved;
    float eps;
    const float *q_norm, *k_norm; /* [head_dim], 16-byte aligned, or NULL */
} q4rdna_kv_append_desc;
int q4rdna_kv_append(const q4rdna_kv_cache *cache, const q4rdna_kv_batch *batch,
                     const q4rdna_kv_append_desc *desc, void *stream);

/* Attention of the step's query tokens, after q4rdna_kv_append of the same
 * batch: out = sum_t softmax_t(scale * q . k_t) v_t over the tokens t <= p of
 * the query's sequence (t > p - window where window > 0), p its position.
 * Query head h reads kv head h / (q_heads / kv_heads).  lse (may be NULL)
 * receives log sum_t exp(scale * q . k_t), [tokens][q_heads].  Calls that
 * split a sequence use scratch per (device, stream), under the rules of the
 * GEMVs' scratch above: make one call of a shape on the stream before
 * capturing it.  Threads may call on one stream at once: no other call's
 * launch that uses the scratch comes between a call's own. */
typedef struct q4rdna_kv_attend_desc {
    uint32_t dtype;           /* of q and out */
    uint32_t q_heads;
    q4rdna_kv_rows q, out;
    float *lse;
    float scale;
    uint32_t window;
} q4rdna_kv_attend_desc;
int q4rdna_kv_attend(const q4rdna_kv_cache *cache, const q4rdna_kv_batch *batch,
                     const q4rdna_kv_attend_desc *desc, void *stream);

/* The cache's tokens past[i] .. past[i] + count - 1 as numbers, in the order of
 * the batch's tokens: k and v [tokens][kv_heads][head_dim] of `dtype`.  The
 * sequence's length must be past[i] + count (its last, open block is found by
 * it); past 0 reads it whole. */
int q4rdna_kv_read(const q4rdna_kv_cache *cache, const q4rdna_kv_batch *batch, uint32_t dtype,
                   const q4rdna_kv_rows *k, const q4rdna_kv_rows *v, void *stream);

/* Residual add with the norms before and after it, per row:
 *   h = residual + scale * gate * post(y)    post(y) = y * rsqrt(mean y^2 + eps) * post_weight, or y
 *   n = h * rsqrt(mean h^2 + eps) * weight
 * y NULL: h = residual.  gate NULL: 1; gate_stride 0: one gate for all rows.
 * post_weight, h and n may be NULL (no norm of y, output not wanted).  n uses
 * h before its rounding to dtype.  h may be residual or y and n may be y or
 * residual, with the same strides; other overlaps are not allowed.  Strides
 * are in elements; width is at most Q4RDNA_NORM_MAX_WIDTH. */
#define Q4RDNA_NORM_MAX_WIDTH 16384
typedef struct q4rdna_add_norm_desc {
    uint32_t dtype;           /* of residual, y, gate, h and n */
    uint32_t rows;
    uint32_t width;
    float scale;
    float eps;
    uint32_t reserved;
    const void *residual, *y, *gate;
    void *h, *n;
    int64_t residual_stride, y_stride, gate_stride, h_stride, n_stride;
    const float *post_weight, *weight; /* [width]; weight may be NULL only where n is */
} q4rdna_add_norm_desc;
int q4rdna_add_norm(const q4rdna_add_norm_desc *desc, void *stream);

/* ---- several continuations of a sequence ------------------------------------
 * Drafted tokens verified together (a tree of them per sequence), beams, and
 * sequences that fork.  No reference counterpart.  As above: asynchronous on
 * `stream`, fp32, fp16 or bf16, sums in fp32 and more. */

/* A sequence of a step has at most so many drafted tokens. */
#define Q4RDNA_TREE_MAX 64

/* Positions and ancestors of a step's drafted tokens, once for all layers.
 * Sequence i has the step's tokens cu_tokens[i] .. (as in q4rdna_kv_batch; of
 * which past, cu_tokens, sequences, tokens and max_tokens <= Q4RDNA_TREE_MAX
 * are used).  parents[n] is the place among its sequence's tokens of token n's
 * parent, which comes before it, or -1 for one that follows the last cached
 * token.  seen[n]: bit j is set where the sequence's j-th token is n itself or
 * above it.  positions[n] = past + the number of tokens above n.  A token whose
 * parent is out of range, those below it, and the tokens of a sequence whose
 * entries are out of range get position -1 and seen 0; tokens of no sequence
 * are not written.  Runs on the current device. */
int q4rdna_kv_tree(const q4rdna_kv_batch *batch, const int32_t *parents, int32_t *positions,
                   uint64_t *seen, void *stream);

/* Rows of q and k normalised and rotated as q4rdna_kv_append does it, bit for
 * bit, by a position given for each token.  A position outside the `positions`
 * rows of cos and sin makes the token's rows NaN.  q_out may be q and k_out k;
 * other overlaps are not allowed.  q_heads or k_heads 0: no q or k.  rotary 0:
 * no rotation, cos, sin and position are not read.  Runs on the current device. */
typedef struct q4rdna_rotate_desc {
    uint32_t dtype;           /* of q, k and the outputs */
    uint32_t tokens;
    uint32_t q_heads, k_heads; /* at most 32768 in all */
    uint32_t head_dim;        /* 64 or 128 */
    uint32_t positions;
    uint32_t rotary;          /* a multiple of 8 up to head_dim */
    uint32_t interleaved;
    q4rdna_kv_rows q, k, q_out, k_out;
    const int32_t *position;  /* [tokens] */
    const float *cos, *sin;   /* [positions][rotary / 2], 16-byte aligned */
    const float *q_norm, *k_norm; /* [head_dim], 16-byte aligned, or NULL */
    float eps;
    uint32_t reserved;
} q4rdna_rotate_desc;
int q4rdna_rotate(const q4rdna_rotate_desc *desc, void *stream);

/* Attention of a step's drafted tokens over the cache and over each other.
 * The drafted tokens are not in the cache: sequence i holds past[i] tokens
 * there, and k and v have the drafted ones' rows (k normalised and rotated).
 * Query token n of a sequence sees the cached tokens and the drafted ones j
 * of its sequence whose bit j is set in seen[n] (q4rdna_kv_tree's, or any
 * other mask):
 *   out = softmax(scale * q . k) v over these, lse as in q4rdna_kv_attend.
 * With window > 0 a drafted token stands at past - 1 + the number of bits in
 * its seen (those of tokens that are there), and sees what lies less than
 * `window` before it: cached tokens at t > p - window, drafted ones at
 * p_j > p - window.
 * A row that sees nothing is zero, its lse -inf.  A drafted token with a number
 * of k (v) that is not finite makes every row that sees it NaN.  Scores are
 * meant to lie within fp32's range: q and k may be of any size.  fp16 and bf16 q,
 * k and v and the cache's codes enter the products as they are, fp32 q, k and v as
 * two fp16 parts, which hold 2^-23 of their row's largest number; weights are held
 * to 2^-22, sums in fp32.
 * The cache is read only; accepted tokens are appended by q4rdna_kv_append of
 * their rows, with rotary 0.  max_tokens <= Q4RDNA_TREE_MAX.  Refusals on the
 * device, and scratch, as for q4rdna_kv_attend. */
typedef struct q4rdna_kv_tree_desc {
    uint32_t dtype;           /* of q, k, v and out */
    uint32_t q_heads;
    q4rdna_kv_rows q, k, v, out;
    const uint64_t *seen;     /* [tokens] */
    float *lse;
    float scale;
    uint32_t window;
} q4rdna_kv_tree_desc;
int q4rdna_kv_attend_tree(const q4rdna_kv_cache *cache, const q4rdna_kv_batch *batch,
                          const q4rdna_kv_tree_desc *desc, void *stream);

/* The best continuations of groups of beams.  For each group, over its beams b
 * and the tokens v of the vocabulary,
 *   total[b][v] = scores[b] + logits[b][v] - log sum_u exp(logits[b][u])
 * and the `count` largest of them, largest first: out_scores, out_rows (group *
 * beams + b) and out_tokens, each [groups][count].  Totals are compared in 64
 * bits; equal ones go by row, then by logit (totals that 64 bits cannot tell
 * apart), then by token.  A beam's log sum comes from fp32 exponentials, added up
 * by 16 in fp32 and then in 64 bits: it is within 2^-18 of the formula's, a few
 * 2^-24 as a rule.  So a beam's own tokens are always in the order of their
 * logits, but totals of two beams that lie closer than that may come either way.
 * scores NULL: zeros.  A beam has no continuation, all its totals are -inf, if
 * its score is not finite, if all its logits are -inf or if one of them is NaN
 * or +inf; such totals come behind all others.  out_scores may be scores where
 * count is beams; other overlaps are not allowed.  Scratch as for
 * q4rdna_kv_attend.  Runs on the current device. */
#define Q4RDNA_BEAM_MAX_COUNT 128
#define Q4RDNA_BEAM_MAX_BEAMS 256
typedef struct q4rdna_beam_desc {
    uint32_t dtype;           /* of logits */
    uint32_t groups;
    uint32_t beams;           /* at most Q4RDNA_BEAM_MAX_BEAMS */
    uint32_t vocab;           /* at most 2^24 */
    uint32_t count;           /* 1 .. Q4RDNA_BEAM_MAX_COUNT, at most beams * vocab */
    uint32_t reserved;
    const void *logits;       /* rows of `vocab` contiguous numbers, strides in elements */
    int64_t group_stride, beam_stride;
    const float *scores;      /* [groups][beams] or NULL */
    float *out_scores;
    int32_t *out_rows, *out_tokens;
} q4rdna_beam_desc;
int q4rdna_beam_select(const q4rdna_beam_desc *desc, void *stream);

/* Sequences that go on from others, in place.  Sequence i of the batch becomes
 * a copy of what sequence parents[i] was: its length, its full pages, which the
 * two share from then on, and its open blocks.  parents[i] = -1: sequence i is
 * dropped, its length becomes 0.
 *  - slots: the first sequence that goes on from a parent takes the parent's
 *    slot, the others the slots of sequences that nobody goes on from, both in
 *    ascending order, and the parent's open blocks are copied there: of a length
 *    m the block m / 64 where it holds tokens, and the one before it.
 *  - table: entries of full blocks come from the parent's row.  A page that is
 *    then in no row's full blocks is free, but for those marked in `kept`, and
 *    the entries of each sequence's open block, where it holds tokens, and of the
 *    blocks that its next `room` tokens touch get free pages (none of a dropped
 *    one): the lowest numbers first, in the order of sequences and blocks.  Other entries become -1, and so do those
 *    that no page is left for, each of which adds to *faults.
 * So `fork` with parents[i] = i gives out the pages for the next tokens, and a
 * program that calls it before each step needs no allocator of its own.  Every
 * sequence that holds pages of these caches has to be in the batch, or its
 * pages in `kept`.  A parent that is out of range, or has a length or a slot
 * that is, drops the sequence, and adds to *faults.  Two sequences may not share
 * a slot.
 * `caches` are the layers' caches, of one geometry (page_count, slot_count,
 * kv_heads, head_dim, device), none of whose buffers may be another's; their
 * pages are neither read nor written.  The batch's past, table and slots are
 * written; cu_tokens, tokens and max_tokens are not used.  Scratch as for
 * q4rdna_kv_attend. */
#define Q4RDNA_FORK_MAX_SEQUENCES 4096
typedef struct q4rdna_kv_fork_desc {
    const int32_t *parents;   /* [sequences] */
    int32_t *past, *table, *slots; /* as in q4rdna_kv_batch, not NULL */
    const uint8_t *kept;      /* [page_count], non-zero: not free, or NULL */
    uint32_t sequences;       /* at most Q4RDNA_FORK_MAX_SEQUENCES */
    uint32_t table_width;
    uint32_t room;
    uint32_t reserved;
} q4rdna_kv_fork_desc;
int q4rdna_kv_fork(const q4rdna_kv_cache *caches, uint32_t count, const q4rdna_kv_fork_desc *desc, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* Q4RDNA_H */
