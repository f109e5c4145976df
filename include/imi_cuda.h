/* imi_cuda.h - C-ABI of the B200 decode engine for imi's brain token loop (the Seoul / LFM3 hybrid backbone).
 *
 * This is the drop-in boundary for imi's brain (reference: imi/core/seoul.h, struct imi_seoul). Plain pointers and
 * sizes only; every call returns an imi_cuda_status and leaves a message for imi_cuda_error(). There is no CPU
 * fallback: without a usable CUDA device every compute call fails with IMI_E_NODEV / IMI_E_CUDA.
 *
 * Model: one engine = one GGUF model resident on one GPU (imi_seoul::load, seoul.cpp:93-186).
 * State: one conversation (attention caches, conv memory, position, latest hidden/logits) resident on the same GPU
 *        (imi_seoul_state, seoul.h:21-26). The engine itself holds no conversation; imi_seoul's "own" conversation is a
 *        state the C++ wrapper (imi_seoul_cuda.h) creates.
 * Step semantics, float order and outputs follow imi_seoul exactly; see each entry point for the reference line. */
#ifndef IMI_CUDA_H
#define IMI_CUDA_H
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct imi_cuda_engine imi_cuda_engine;
typedef struct imi_cuda_state imi_cuda_state;

typedef enum {
    IMI_OK = 0,
    IMI_E_ARG = 1,       /* bad argument (null pointer, token out of range, n <= 0, states of another engine) */
    IMI_E_FILE = 2,      /* GGUF file missing or unreadable (imi: load() returns false, seoul.cpp:94) */
    IMI_E_FORMAT = 3,    /* a tensor is missing or has a type/shape the kernels do not read (seoul.cpp:96,162) */
    IMI_E_CTX_FULL = 4,  /* position would pass n_ctx: nothing is stepped (imi prints "context full", seoul.cpp:353) */
    IMI_E_CUDA = 5,      /* a CUDA call failed */
    IMI_E_NOMEM = 6,     /* device (or pinned host) allocation failed */
    IMI_E_TIMEOUT = 7,   /* a bounded device-side wait gave up (the kernel returned; the context stays usable) */
    IMI_E_NODEV = 8      /* no CUDA device with the requested index */
} imi_cuda_status;

typedef struct {
    int n_embd, n_vocab, n_ctx, n_layer, n_attn, n_head, n_head_kv, head_dim, n_ff, d_conv, n_swa, max_batch;
    size_t weight_bytes;   /* bytes of layer tables + word table + small parameters on the device */
    size_t state_bytes;    /* device bytes of one conversation state */
    int cols_per_read;     /* conversations (or prefill positions) one read of the tables serves at most: 8 on the
                              small-batch kernel; up to 256 (max(max_batch, 128)) on the tensor cores, which every
                              Q4_0 model uses above 8 */
} imi_cuda_info;

/* Last error message of this thread (never NULL). */
const char *imi_cuda_error(void);

/* Load a GGUF model onto CUDA device `device` (replaces imi_seoul::load(path, threads, ctx_len), seoul.cpp:93).
 * n_ctx: positions per conversation; max_batch: most conversations stepped together by imi_cuda_step_multi.
 * An engine and its states are used by one host thread at a time: they share the engine's stream, its staging
 * buffers and its read-back buffer.
 * Device memory budget: when the environment variable IMI_CUDA_MAX_DEVICE_BYTES is set (bytes), the engine and all
 * its states together allocate at most that much; a load or a new state beyond it fails with IMI_E_NOMEM (for a GPU
 * shared with other work). */
imi_cuda_status imi_cuda_load(const char *gguf_path, int device, int n_ctx, int max_batch, imi_cuda_engine **out);
void imi_cuda_free(imi_cuda_engine *e);                                     /* ~imi_seoul, seoul.cpp:687-689 */
imi_cuda_status imi_cuda_get_info(const imi_cuda_engine *e, imi_cuda_info *out);

/* A fresh conversation sized like the engine's (imi_seoul::new_state, seoul.cpp:193-201): position 0, zero conv memory. */
imi_cuda_status imi_cuda_state_new(imi_cuda_engine *e, imi_cuda_state **out);
void imi_cuda_state_free(imi_cuda_state *s);
/* Position 0 and zero conv memory (imi_seoul::reset, seoul.cpp:188-191). */
imi_cuda_status imi_cuda_state_reset(imi_cuda_state *s);
int imi_cuda_state_pos(const imi_cuda_state *s);                            /* imi_seoul::pos */

/* One position (imi_seoul::step, seoul.cpp:352-357): token >= 0 reads the word table row, else embd[n_embd] is the
 * input vector. want_logits adds the word scores (and the greedy pick). IMI_E_CTX_FULL if pos >= n_ctx. */
imi_cuda_status imi_cuda_step(imi_cuda_state *s, int32_t token, const float *embd, int want_logits);

/* Two conversations one position each, every table read once for both (imi_seoul::step2, seoul.cpp:208-220).
 * Each gets exactly the numbers its own imi_cuda_step would give. */
imi_cuda_status imi_cuda_step2(imi_cuda_state *a, int32_t token_a, const float *embd_a, int logits_a,
                               imi_cuda_state *b, int32_t token_b, const float *embd_b, int logits_b);

/* n distinct conversations of one engine, one position each, one table read for all (n <= max_batch): the
 * generalisation of step2 to the multi-session case. tokens[i] (or embd + i*n_embd when tokens is NULL or
 * tokens[i] < 0), want_logits[i] (NULL = all). */
imi_cuda_status imi_cuda_step_multi(imi_cuda_state *const *s, int n, const int32_t *tokens, const float *embd,
                                    const int *want_logits);

/* Read n positions of one conversation (imi_seoul::step_batch, seoul.cpp:490-517): tokens[n], or embd[n][n_embd].
 * hidden and (if want_logits) logits are the last position's; hidden_all[n][n_embd] (host, optional) receives every
 * position's hidden state. Positions are read in chunks; IMI_E_CTX_FULL (nothing more stepped) when a chunk would
 * pass n_ctx, as seoul.cpp:498. */
imi_cuda_status imi_cuda_step_batch(imi_cuda_state *s, const int32_t *tokens, const float *embd, int n,
                                    int want_logits, float *hidden_all);

/* Greedy decode on the device: `steps` positions for each of n conversations (n <= max(max_batch, 8)), each step's
 * input being the previous step's pick (the caller loop of imi/core/hear.cpp:65-72 without a stop word). The first
 * step reads tokens[i] (or, when tokens is NULL, each conversation's last pick). ids[steps][n] receives every pick.
 * Logits of the last step stay readable. */
imi_cuda_status imi_cuda_greedy(imi_cuda_state *const *s, int n, const int32_t *tokens, int steps, int32_t *ids);

/* Sampling from conversations' latest word scores (imi picks greedily only): the words imi_cuda_sample (below) names for the
 * uniform numbers u[n], with per-conversation settings (arrays of n, host; NULL: temperature 1, the filters off). ids,
 * logprob and kept (each may be NULL) receive them. A word becomes its conversation's last pick: what imi_cuda_get_argmax
 * returns, with its score, and what a later imi_cuda_greedy or imi_cuda_sampled without tokens reads first. */
imi_cuda_status imi_cuda_sample_states(imi_cuda_state *const *s, int n, const float *u, const float *temperature,
                                       const int32_t *top_k, const float *top_p, const float *min_p, int32_t *ids, float *logprob,
                                       int32_t *kept);

/* imi_cuda_greedy with sampling: `steps` positions for each of n conversations, each step's input being the word sampled
 * after the step before (the first: tokens[i], or the conversation's last pick when tokens is NULL). u[steps][n] (host): the
 * uniform number of each word; settings as above, the same for all steps. ids[steps][n] and logprob[steps][n] may be NULL.
 * Temperature 0 gives what imi_cuda_greedy gives. The words stay on the device from step to step. */
imi_cuda_status imi_cuda_sampled(imi_cuda_state *const *s, int n, const int32_t *tokens, int steps, const float *u,
                                 const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                                 int32_t *ids, float *logprob);

/* A conversation's cached keys and values of one attention layer (0..n_attn-1), on the device: IMI_F16, position p of kv
 * head h at k + p * position_stride + h * head_stride (elements; v alike), positions 0..pos-1. Keys are normed and rotated
 * as the engine's attention reads them. For imi_cuda_page_write: a prompt the engine has read, into pages. The pointers
 * stay the conversation's; its steps write further positions on the engine's stream (imi_cuda_stream), so a reader on
 * another stream waits for that. */
imi_cuda_status imi_cuda_state_kv(const imi_cuda_state *s, int layer, const void **k, const void **v, int64_t *position_stride,
                                  int64_t *head_stride);

/* Checkpoint / resume of one conversation (the content of imi_seoul_state, seoul.h:21-26) as a host byte image:
 *   int32 magic 0x53494d49 ("IMIS"), version 1, pos, n_attn, n_ctx, kv_dim, n_conv, d_conv, n_embd, n_vocab, next_pick;
 *   K cache [n_attn][pos][kv_dim] fp16, V cache likewise (positions 0..pos-1 only);
 *   conv memory [n_conv][d_conv][n_embd] fp32, oldest first (imi's layout, seoul.h:47);
 *   hidden [n_embd] fp32, logits [n_vocab] fp32.
 * save: buf NULL -> *size receives the bytes needed; else the image is written (cap >= that size).
 * load: into a state of an engine with the same shape and an n_ctx >= the image's pos. */
imi_cuda_status imi_cuda_state_save(const imi_cuda_state *s, void *buf, size_t cap, size_t *size);
imi_cuda_status imi_cuda_state_load(imi_cuda_state *s, const void *buf, size_t size);

/* The latest outputs of a conversation (imi_seoul::hidden / ::logits, seoul.h:51): host copies. */
imi_cuda_status imi_cuda_get_hidden(const imi_cuda_state *s, float *out /* n_embd */);
imi_cuda_status imi_cuda_get_logits(const imi_cuda_state *s, float *out /* n_vocab */);
/* The greedy pick of the latest step with logits: first maximum, lowest id on ties (imi/core/hear.cpp:67-68); or the word
 * sampled since (imi_cuda_sample_states, imi_cuda_sampled). value (may be NULL): its score (0 behind imi_cuda_state_load,
 * whose image does not hold it). */
imi_cuda_status imi_cuda_get_argmax(const imi_cuda_state *s, int32_t *id, float *value);

/* ---- the model file's keys and tensor headers (host only; imi_file, imi/model.h:17-36) ----
 * The GGUF file memory-mapped by the library's own reader, for callers that read keys beside the brain (the
 * tokenizer reads the word list from the same file: imi_words::load(brain.f), flow.cpp:49). Value types are GGUF's
 * (4 u32, 5 i32, 6 f32, 7 bool, 8 string, 9 array, 10 u64, ...). Pointers stay valid until imi_cuda_file_close. */
typedef struct imi_cuda_file imi_cuda_file;
imi_cuda_status imi_cuda_file_open(const char *path, imi_cuda_file **out);
void imi_cuda_file_close(imi_cuda_file *f);
int64_t imi_cuda_file_find_key(const imi_cuda_file *f, const char *key);              /* -1 when absent */
int64_t imi_cuda_file_n_keys(const imi_cuda_file *f);
const char *imi_cuda_file_key_name(const imi_cuda_file *f, int64_t k);
int imi_cuda_file_key_type(const imi_cuda_file *f, int64_t k);
const void *imi_cuda_file_key_data(const imi_cuda_file *f, int64_t k);                  /* a scalar's bytes */
const char *imi_cuda_file_key_str(const imi_cuda_file *f, int64_t k);                   /* a string (copy, 0-ended) */
int imi_cuda_file_arr_type(const imi_cuda_file *f, int64_t k);
uint64_t imi_cuda_file_arr_n(const imi_cuda_file *f, int64_t k);
const void *imi_cuda_file_arr_data(const imi_cuda_file *f, int64_t k);                  /* fixed-size elements */
const char *imi_cuda_file_arr_str(const imi_cuda_file *f, int64_t k, uint64_t i);       /* string element i */
/* a tensor's header: 0 and its GGML type, shape (fastest first), bytes in the map; -1 when absent */
int imi_cuda_file_tensor(const imi_cuda_file *f, const char *name, int *type, int64_t ne[4], const void **data,
                         size_t *nbytes);

/* ---- measurement ---- */

/* The CUDA stream (cudaStream_t) every launch of this engine goes to, for callers that time on the device. */
void *imi_cuda_stream(const imi_cuda_engine *e);
/* Milliseconds on the device of the engine's last step (the last read of its tables with everything around it:
 * every launch of one imi_cuda_step / step2 / step_multi group / step_batch chunk), waiting for it to finish; 0 if
 * none ran. The C++ wrapper adds it to imi_seoul::t_tables after each step. */
float imi_cuda_last_step_ms(const imi_cuda_engine *e);
/* Kernel launches of one step of n conversations (with or without word scores). */
int imi_cuda_launches_per_step(const imi_cuda_engine *e, int n, int want_logits);
/* Kernel launches of one imi_cuda_step_batch of n positions (with or without the last position's word scores). */
int imi_cuda_launches_per_batch(const imi_cuda_engine *e, int n, int want_logits);
/* Every layer table read back to back with ncol (1..cols_per_read) inputs riding each read, as imi_seoul::bench_tables
 * (seoul.cpp:657-685): *ms = mean milliseconds per pass over `reps` passes (after one untimed pass), *bytes = table
 * bytes read per pass. */
imi_cuda_status imi_cuda_bench_tables(imi_cuda_engine *e, int ncol, int reps, float *ms, size_t *bytes);

/* Diagnostics: read table `which` (0 in_proj/qkvg, 1 out_proj/o, 2 gate_up, 3 down) of layer `layer`
 * once, alone, with ncol inputs, and return per-CTA phase timestamps in ns: trace[cta][16] (0 start, 1 after the
 * dependency wait, 2 after input preparation, 3+s after stage s's integer phase, 14 end of the float chains).
 * *grid receives the number of CTAs; trace must hold 148*16 values on a B200. */
imi_cuda_status imi_cuda_trace_table(imi_cuda_engine *e, int layer, int which, int ncol, unsigned long long *trace,
                                     int *grid);

/* Diagnostics: one decode step of `s` (token given) launched directly (not from a graph) with every launch writing
 * per-CTA phase timestamps (ns): out[launch][n_sm][16] as in imi_cuda_trace_table (final norm: 0 start, 1 after the
 * dependency wait, 14 end; attention at head_dim 64 adds 2 query and this position's K/V made, 3 scores, 4
 * probabilities, 5 P.V done, 6 the first K/V copies issued, 7 / 8 the first / last K tile landed, 9 / 10 the first /
 * last V tile landed). kinds[launch]: 10*input+output kind of a table read, 100 attention, 101 final norm;
 * grids[launch]: CTAs. *n receives the number of launches (at most max_launches). */
imi_cuda_status imi_cuda_trace_step(imi_cuda_state *s, int32_t token, int want_logits, unsigned long long *out,
                                    int max_launches, int *kinds, int *grids, int *n);

/* Diagnostics: the failure path of the engine's bounded device waits (every wait on a weight stage gives up after
 * about one second and reports IMI_E_TIMEOUT instead of hanging). One CTA waits on an mbarrier that nothing completes,
 * with a limit of limit_ms milliseconds at the device's clock; the wait gives up, the kernel sets the error flag and
 * returns. Returns IMI_E_TIMEOUT when the wait gave up as designed (the context stays usable), IMI_OK never. */
imi_cuda_status imi_cuda_check_wait_timeout(int device, double limit_ms);

/* ---- kernel level (known-answer tests and the isolated table sweep) ---- */

/* Cut x[n] to 8-bit per 32 values on the device (imi_q8::from, tables.cpp:100-109 with imi_cut32, vec.h:47-77):
 * q[n] int8 codes, d[n/32] scales, s[n/32] = d * sum(q). Host pointers. */
imi_cuda_status imi_cuda_q8_cut(int device, const float *x, int n, int8_t *q, float *d, float *s);

/* Word scores of a Q6_K table (the product's own word-table format: rows of 210-byte blocks per 256 values) for one
 * float input x[cols], on the device: the input cut per 256 values as imi_q8k::from (tables.cpp:200-213), then every
 * row as imi_q6k_row (tables.cpp:235-278, the AVX2 order) -> out[rows]. The cut can be returned too (xq[cols],
 * xd[cols/256], bsums[cols/16]; each may be NULL). cols a multiple of 256, at most 32768; host pointers. The kernel
 * level of the Q6_K word table, which the engine also reads inside its steps when a file carries one. */
imi_cuda_status imi_cuda_q6k_scores(int device, const uint8_t *q6k, int rows, int cols, const float *x, float *out,
                                    int8_t *xq, float *xd, int16_t *bsums);

/* A Q4_0 table (GGUF rows of 18-byte blocks, rows x cols) times ncol 8-bit inputs (xq[ncol][cols], xd/xs[ncol][cols/32])
 * on the device with imi's 4-bit kernel semantics (imi_q4_group / imi_q4_group2 / imi_q4_group_batch,
 * tables.cpp:127-177,419-477): out[ncol][rows]. Host pointers; block_dots (optional, ncol == 1) receives the integer
 * dot of every (row, 32-block) pair [rows][cols/32]. */
imi_cuda_status imi_cuda_q4_matvec(int device, const uint8_t *q4, int rows, int cols, const int8_t *xq,
                                   const float *xd, const float *xs, int ncol, float *out, int32_t *block_dots);

/* The same table read for many inputs on the tensor cores (the batched read of imi_q8b + imi_q4_group_batch,
 * tables.cpp:405-477): ncol 1..256 inputs, each block's integer dot by a tcgen05 MMA (8-bit codes, int32, exact), imi's float
 * chains per (row, input) in block order; results as imi_cuda_q4_matvec gives them. Host pointers. */
imi_cuda_status imi_cuda_q4_matmul(int device, const uint8_t *q4, int rows, int cols, const int8_t *xq,
                                   const float *xd, const float *xs, int ncol, float *out);

/* Diagnostics: imi_cuda_q4_matmul with CTA 0's timeline of the tensor-core read in ns, trace[9][64]: 0 stage copies
 * issued, 1 (unused, 0), 2 stage done by the last epilogue warp, 3 block's MMA issued, 4 block's dots awaited by the
 * epilogue, 5 block's chains done, 6 block's dots in registers, 7 stage's copies seen by the MMA warp, 8 stage's TMEM
 * slot free for the MMA warp (stages and blocks counted from the CTA's first unit); trace holds 9 * 64 values. */
imi_cuda_status imi_cuda_trace_tc(int device, const uint8_t *q4, int rows, int cols, const int8_t *xq, const float *xd,
                                  const float *xs, int ncol, float *out, unsigned long long *trace);

/* The isolated table read timed on the device (the configs[4] sweep; imi/kernels/q4x2_bench.cpp's measurement): a
 * rows x cols Q4_0 table (random codes and scales, the engine's row layout) times ncol 8-bit inputs, `reps` reads after
 * one untimed pass, CUDA events on one stream. The table is replicated in device memory until the copies pass 256 MB
 * and the reads rotate through all of them (at least `reps` reads, at least one per copy), so every read comes from
 * HBM (L2 holds 126 MB). *ms = mean milliseconds per
 * read of all ncol inputs; *bytes = algorithmic bytes per read: the table once, the inputs' codes and scales, the
 * outputs. ncol 1..256; cols a multiple of 256. */
imi_cuda_status imi_cuda_bench_matvec(int device, int rows, int cols, int ncol, int reps, float *ms, size_t *bytes);

/* ---- without allocation ---- */

/* No counterpart in the reference (imi's own path has no device memory): imi_cuda_q4_matvec on device buffers that
 * allocates nothing. It exists for callers that must not allocate device memory while they run: cudaFree waits for
 * every stream of the device (a caller sharing the GPU with a running decode loop would stall it), a cudaMalloc may
 * fail once a memory pool or another framework's caching allocator holds the free memory, and some callers run where
 * allocating is not allowed at all (a real-time audio callback, an allocator hook).
 *
 * q4: the table as GGUF Q4_0 rows (rows x cols, 18-byte blocks); xq[ncol][cols] (16-byte aligned), xd, xs[ncol][cols/32]
 * and out[ncol][rows]: all device memory of `device`; results as imi_cuda_q4_matvec gives them. stream: a cudaStream_t
 * of that device (NULL: the default stream); the call returns once its work on that stream is done.
 * Scratch: one static device array of this library per device (IMI_CUDA_STATIC_TABLE_BYTES for the table in the
 * kernels' row layout, plus 4 KiB). The call clears what must start at zero (the column descriptors and the error
 * flag) on the stream itself, so nothing needs to be zero beforehand. A table above IMI_CUDA_STATIC_TABLE_BYTES
 * (rows * cols / 32 * 18 bytes) is refused with IMI_E_ARG.
 * The first call on a device looks the scratch address up (cudaGetSymbolAddress, with that device current) and sets
 * the kernels' shared-memory limits; both are kept for the life of the process, which assumes the device's primary
 * context is not reset (cudaDeviceReset) in between. The scratch is shared: two calls on the same device that overlap in time (from two host threads,
 * or on two streams) race on it and corrupt each other's results; callers serialise them. */
#define IMI_CUDA_STATIC_TABLE_BYTES 16777216u
imi_cuda_status imi_cuda_q4_matvec_static(int device, const uint8_t *q4, int rows, int cols, const int8_t *xq,
                                          const float *xd, const float *xs, int ncol, float *out, void *stream);

/* ---- serving operators on device buffers ----
 *
 * No counterpart in the reference (imi serves a handful of conversations, each with its own contiguous memory, and picks
 * greedily): what a server of many conversations on one GPU needs beside the step, as operators a caller runs on buffers
 * of its own: pages instead of one n_ctx-sized cache per conversation, attention that reads a prompt all conversations
 * share once for all of them, and sampling.
 *
 * In common: every pointer in the argument blocks is device memory of `device` (checked; IMI_E_ARG otherwise), unless it
 * is said to be optional and is NULL. A call checks its arguments on the host, enqueues its kernels on `stream` (a
 * cudaStream_t of that device; NULL: the default stream) and returns without waiting; it allocates nothing and may be
 * captured into a CUDA graph, which then replays with the same pointers and sizes and whatever the buffers hold. The
 * current device of the calling thread is left as it was. Calls from several threads or on several streams are
 * independent as long as they write different buffers (outputs, workspaces and status words included).
 * What only the device can see (lengths, page numbers, slots) is checked there: nothing outside the buffers is read or
 * written, and the largest IMI_DEV_* code met is left in the call's status word (atomic maximum; a call never clears
 * it: the caller zeroes it when it has read it). Where a call takes no status word, what it met is not reported. */
typedef enum { IMI_F32 = 0, IMI_F16 = 1, IMI_BF16 = 2 } imi_cuda_type;
enum {
    IMI_DEV_PAGE = 1,    /* a page number outside 0..n_pages-1, or a slot beyond the last page */
    IMI_DEV_TABLE = 2,   /* a request longer than its block table's row holds */
    IMI_DEV_CAP = 3,     /* the step's new positions exceed the slot arrays */
    IMI_DEV_POOL = 4,    /* not enough free pages (or a free count outside the list) */
    IMI_DEV_LENGTH = 5,  /* a negative number of new positions */
    IMI_DEV_WAIT = 6     /* a bounded device-side wait gave up (the call's outputs are not usable) */
};

/* Block tables and slot maps from the requests' lengths.
 * Request i holds held[i] positions and adds add[i]; its pages are table[i * table_stride + c], c counting pages of
 * `page` positions (a power of two, 16..256). Pages it lacks are taken from the end of the free list (a stack: page
 * k-th taken is free_pages[n_free - 1 - k]), request by request, and entered into its row; nothing else of the table
 * is written. held[i] < 0 marks a row that is not in use (add ignored, length -1).
 *   start[n + 1]   exclusive sums of add: request i's new positions are rows start[i]..start[i+1]-1 of the step
 *   length[n]      held + add
 *   slots[cap]     per new row: page number * page + offset in the page; -1 behind the last
 *   pos[cap]       per new row: its position, pos0 + (position within the request's own pages); -1 behind the last
 *   n_free_out[1]  free pages left (the list itself is not written)
 * length may be held's buffer, n_free_out may be n_free's (the next step's inputs in place). When a request passes
 * its table row (IMI_DEV_TABLE), the new rows exceed cap, the pool is short or a length is negative, the step maps
 * nothing: slots and pos are -1 throughout, start 0, length = held, n_free_out = n_free, the table as it was. A page
 * number outside the pool (IMI_DEV_PAGE) makes its slots -1. status[2]: the status word, then a counter that must be 0
 * before the first call and is 0 after every call; calls that share status run one after the other. n <= 4096. */
typedef struct {
    const int32_t *held, *add;
    int n;
    int32_t *table;
    int64_t table_stride;
    int width;                      /* pages per table row */
    const int32_t *free_pages;
    int free_cap;                   /* entries of free_pages (0: none) */
    const int32_t *n_free;
    int page, n_pages, pos0, cap;
    int32_t *start, *length, *slots, *pos, *n_free_out, *status;
} imi_cuda_page_map_args;
imi_cuda_status imi_cuda_page_map(int device, const imi_cuda_page_map_args *a, void *stream);

/* K and V rows into pages: row r, head h of k (k + r * row_stride + h * head_stride, in elements; v alike) goes to
 * offset slots[r] % page of page slots[r] / page of k_pages, [n_pages][n_head_kv][page][head_dim] (v_pages alike),
 * rounded to nearest even where the pages' type is narrower. slots[r] < 0: row r is skipped. head_dim a multiple of 8,
 * at most 256; pages IMI_F16 or IMI_BF16, rows those of the pages' type or IMI_F32; pages 16-byte aligned (rows of any
 * alignment; 16-byte aligned ones with strides of whole 16 bytes are read in 16-byte pieces). Slots of one call are
 * distinct, as imi_cuda_page_map makes them: of rows with the same slot each element is one of theirs. status optional. */
typedef struct {
    const void *k, *v;
    int type;                       /* imi_cuda_type of the rows */
    int64_t row_stride, head_stride;
    int rows;
    const int32_t *slots;
    int n_head_kv, head_dim;
    void *k_pages, *v_pages;
    int page_type, page, n_pages;
    int32_t *status;
} imi_cuda_page_write_args;
imi_cuda_status imi_cuda_page_write(int device, const imi_cuda_page_write_args *a, void *stream);

/* Attention of one new token per conversation over a prompt that all of them share and the conversation's own pages.
 * Conversation i sees the prompt's prefix_len positions (the pages prefix[0..], in order, the last one possibly in part)
 * and then its own length[i] positions (pages table[i * table_stride + c]); with window > 0 only the last `window` of
 * these prefix_len + length[i] positions (the engine's sliding-window layers: the query's own position included).
 *   out[i][h] = sum_j p_j V_j,  p = softmax(scale * q[i][h] . K_j),  lse[i][h] = log sum_j exp(scale * q . K_j)
 * Head h reads kv head h / (n_head / n_head_kv). The prompt's pages are read once for the whole batch. A conversation
 * that sees nothing gets out 0 and lse -infinity. length[i] < 0: the row is not in use, its out and lse stay as they
 * were. A score of NaN or +infinity at a position that a conversation sees makes its out and lse NaN. Positions beyond a
 * length may hold anything, NaN included; a NaN or infinity in V at a prompt position that some conversation's window
 * includes may reach the others' outputs too.
 * type: IMI_F16 or IMI_BF16, of q and the pages; products, softmax and sums are held in 32 bits, the probabilities
 * rounded to `type` for their product with V. scale * log2(e) is finite. out_type: any imi_cuda_type. head_dim 64 or
 * 128; n_head / n_head_kv at most 16; rows at most 4096; page a power of two, 16..256; the prompt and a table row together
 * at most 2^30 - page positions, all table rows below 2^35; q and pages 16-byte aligned, q's and out's rows q_stride /
 * out_stride elements apart (multiples of 8), heads head_dim apart. A length beyond its table row
 * (IMI_DEV_TABLE) counts as the row's positions; a page number outside the pool (IMI_DEV_PAGE) hides its positions.
 * The call is planned from width, not from the lengths: a width near the longest own length serves it best (table_stride
 * may be larger; a workspace for a larger width fits).
 * work: imi_cuda_prefix_attn_work(...) bytes, 16-byte aligned, nothing expected in it; calls that may overlap need one
 * each. lse and status optional. */
typedef struct {
    const void *q;
    int type;
    int64_t q_stride;
    int rows, n_head, n_head_kv, head_dim;
    const void *k_pages, *v_pages;
    int page, n_pages;
    const int32_t *prefix;
    int prefix_len;
    const int32_t *table;
    int64_t table_stride;
    int width;                      /* pages per table row (0: no own pages) */
    const int32_t *length;
    float scale;
    int window;
    void *out;
    int out_type;
    int64_t out_stride;
    float *lse;
    void *work;
    size_t work_bytes;
    int32_t *status;
} imi_cuda_prefix_attn_args;
/* workspace bytes of a call of at most these sizes (smaller ones of the same heads fit) */
size_t imi_cuda_prefix_attn_work(int rows, int n_head, int n_head_kv, int head_dim, int prefix_len, int width, int page);
imi_cuda_status imi_cuda_prefix_attn(int device, const imi_cuda_prefix_attn_args *a, void *stream);

/* A word per row of scores[n][vocab] (rows `stride` elements apart, any imi_cuda_type) from a given uniform number u[i]
 * in [0, 1). With x the row's scores, w_j = exp((x_j - max x) / temperature), words ordered by score, equal scores by id:
 *   top-k  the first top_k words (0 or less: all)
 *   top-p  of those, the words before which less than top_p of their total weight lies (1 or more, or NaN: all); the
 *          first always
 *   min-p  of those, the words of w_j >= min_p (0 or less, or NaN: all); the first always
 * ids[i] is the first word, by id, at which the running sum of the kept weights exceeds u[i] times their total;
 * logprob[i] = log(its weight / that total); kept[i] the number of words kept. temperature 0 (or negative, or NaN):
 * the greedy pick (highest score, lowest id), logprob 0, kept 1, as imi_cuda_get_argmax. Words of score -infinity or NaN are
 * never kept; a row of nothing else gives id -1, logprob -infinity, kept 0. Scores of +infinity share the row evenly.
 * Weights are exact to 2^-44 of the largest word's and summed as integers: the word does not depend on the order of
 * the sums. Per-row settings (temperature, top_k, top_p, min_p) are optional; without them 1, 0, 1, 0.
 * vocab at most IMI_CUDA_SAMPLE_VOCAB. logprob and kept optional. */
#define IMI_CUDA_SAMPLE_VOCAB 262144
typedef struct {
    const void *scores;
    int type;
    int64_t stride;
    int n, vocab;
    const float *u, *temperature;
    const int32_t *top_k;
    const float *top_p, *min_p;
    int32_t *ids;
    float *logprob;
    int32_t *kept;
} imi_cuda_sample_args;
imi_cuda_status imi_cuda_sample(int device, const imi_cuda_sample_args *a, void *stream);

#ifdef __cplusplus
}
#endif
#endif
