/*
 * qe.h -- C ABI of the MI355X-native Qwen3 batch-1 decode engine (libqe.so).
 *
 * The engine API of the reference's Rust crate, flattened to plain C so that a Rust `-sys`
 * crate (or ctypes, or C++) can bind it without any GPU types in the signatures. Every entry
 * point returns an int status (QE_OK == 0) and never aborts; qe_last_error() gives the message
 * of the last failure on the calling thread. A model handle and the caches made from it are
 * single-threaded: calls on one model must not overlap (the reference's MetalModel shares its
 * scratch buffers the same way, metal_inference.rs:85-98).
 *
 * Reference interfaces replaced (paths relative to the reference root):
 *   metal_infrence_engine/src/cpu_inference.rs, metal_infrence_engine/src/metal_inference.rs,
 *   metal_infrence_engine/src/bin/bench.rs, metal_infrence_engine/tests/read_bandwidth.rs.
 */
#ifndef QE_H
#define QE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* status codes */
#define QE_OK 0
#define QE_ERR_IO 1          /* file missing or unreadable (io::Error in the reference) */
#define QE_ERR_FORMAT 2      /* bad safetensors header / config.json / alignment */
#define QE_ERR_TENSOR 3      /* missing tensor, non-BF16 dtype, or shape mismatch */
#define QE_ERR_POS 4         /* pos >= max_seq, or pos beyond the cached length */
#define QE_ERR_ARG 5         /* invalid argument (null pointer, token >= vocab, ...) */
#define QE_ERR_UNSUPPORTED 6 /* a shape the kernels do not handle (head_dim != 128, ...) */
#define QE_ERR_HIP 7         /* a HIP runtime call failed */
#define QE_ERR_NO_DEVICE 8   /* no usable gfx950 device */
#define QE_ERR_KERNEL 9      /* a kernel reported a failure through its error word */

/* KV cache element types */
#define QE_KV_F32 0
#define QE_KV_BF16 1
#define QE_KV_FP8 2 /* e4m3 with a power-of-two scale per row: pages only (qe_pages) */

/* Subset of config.json the forward pass reads. Replaces `Config`, cpu_inference.rs:20-33. */
typedef struct qe_config {
  uint64_t hidden_size;
  uint64_t intermediate_size;
  uint64_t num_hidden_layers;
  uint64_t num_attention_heads;
  uint64_t num_key_value_heads;
  uint64_t head_dim;
  uint64_t vocab_size;
  float rms_norm_eps;
  float rope_theta;
  uint32_t eos_token_id;
} qe_config;

typedef struct qe_model qe_model;
typedef struct qe_kv qe_kv;

/* Called once per finished decode step with that step's greedy token, in order. */
typedef void (*qe_on_token)(void* user, uint32_t token);

/* Message of the last failed call on this thread ("" if none). Valid until the next call. */
const char* qe_last_error(void);

/* ---- model: MetalModel::load_model (metal_inference.rs:157-168), which reads the file with
 *      Model::load_model (cpu_inference.rs:58-84) and the sibling config.json. Weights are
 *      copied once into a device arena on the current HIP device. ---- */
int qe_model_load(const char* safetensors_path, qe_model** out);
void qe_model_free(qe_model* model);
/* MetalModel::config (metal_inference.rs:170) */
int qe_model_config(const qe_model* model, qe_config* out);
/* The HIP stream (hipStream_t) every call on this model is ordered on, so a caller can time
 * it with its own events. No reference counterpart: the Metal engine keeps its queue private. */
void* qe_model_stream(const qe_model* model);
/* bench.rs:106-116 (tests/mbu.rs:19-30): every tensor's bytes except the embedding table,
 * plus one embedding row */
uint64_t qe_weight_bytes_per_token(const qe_model* model);
/* bench.rs:118-119: K and V bytes read at position pos (f32 as in the reference; bf16 halves) */
uint64_t qe_kv_bytes_at(const qe_model* model, uint64_t pos, int kv_dtype);
/* How this model's decode step runs its layers: 2 = all of them in one persistent launch, 1 = two
 * launches per layer (attention block, MLP block), 0 = one launch per stage. 1 and 2 serve one KV
 * head per XCD and need the Qwen3-0.6B shape on a device that deals a launch's workgroups to its
 * XCDs round-robin; QE_FUSED=0, 1 or 2 at model load caps the choice. No reference counterpart:
 * the Metal engine encodes one dispatch per stage (metal_inference.rs:318-387). */
int qe_model_fused_layers(const qe_model* model);

/* ---- KV cache: MetalKVCache::new (metal_inference.rs:129-137). One cache per sequence,
 *      tied to the model it was made from; holds the RoPE table for max_seq positions. ---- */
int qe_kv_new(qe_model* model, uint64_t max_seq, int kv_dtype, qe_kv** out);
void qe_kv_free(qe_kv* kv);
uint64_t qe_kv_max_seq(const qe_kv* kv);
/* positions cached so far (the next forward must use pos <= this) */
uint64_t qe_kv_len(const qe_kv* kv);

/* ---- one token: MetalModel::forward (metal_inference.rs:284-291) == Model::forward
 *      (cpu_inference.rs:98-179). Runs `token` at `pos`, writes its K/V into the cache and
 *      returns the vocab_size logits in logits_out (host memory). Requires pos < max_seq and
 *      pos <= qe_kv_len(kv); afterwards qe_kv_len(kv) == pos + 1. ---- */
int qe_forward(qe_model* model, uint32_t token, uint64_t pos, qe_kv* kv, float* logits_out);

/* ---- prefill: the prompt loop of bench.rs:174-176 (one forward per token). Writes the last
 *      position's logits to last_logits (nullable). n = 0 does nothing: last_logits and the
 *      cache are left as they were. ---- */
int qe_prefill(qe_model* model, const uint32_t* ids, uint64_t n, uint64_t start_pos, qe_kv* kv,
               float* last_logits);

/* ---- greedy decode: MetalModel::decode (metal_inference.rs:293-316). `first` goes in at
 *      start_pos; each step's GPU argmax (lowest index on ties, main.rs:37-42) feeds the next
 *      step on the device. on_token (nullable) is called with each step's token as the step
 *      finishes. If logits_per_step is not NULL it receives steps*vocab_size floats (slower:
 *      one device-to-host copy per step; meant for parity tests). steps = 0 does nothing. ---- */
int qe_decode(qe_model* model, uint32_t first, uint64_t start_pos, uint64_t steps, qe_kv* kv,
              qe_on_token on_token, void* user, float* logits_per_step);

/* ---- multi-token forward on the matrix cores (no reference counterpart: the reference's
 *      prompt loop calls forward once per token, bench.rs:174-176) ---- */
/* Chunked prefill: runs ids[0..n) at positions start_pos.. through the model in chunks of up to
 * `chunk` tokens (0 = 512, at most 2048): one bf16 MFMA GEMM per projection and chunk, f32
 * activations split into two bf16 halves (about 16 mantissa bits), causal attention over the
 * cache and the chunk. Appends the K/V of every position and writes the last token's logits
 * (nullable). Same position contract as qe_prefill; logits agree with it within 1e-2, not bit for
 * bit. The model's chunk buffers are allocated on first use. Consecutive chunks of more than 32
 * tokens run on two streams (the model's and one it creates on first use, with a second set of
 * chunk buffers), each chunk's attention ordered after the earlier chunks' K/V rows of the same
 * layer; the call returns once every stream is done. n = 0 does nothing. */
int qe_prefill_batch(qe_model* model, const uint32_t* ids, uint64_t n, uint64_t start_pos, qe_kv* kv,
                     uint32_t chunk, float* last_logits);
/* Verify k (1..64) tokens at positions start_pos.. in one pass (the k-token check of speculative
 * decoding): appends their K/V and writes all k logit rows, logits_out [k][vocab_size]. */
int qe_verify(qe_model* model, const uint32_t* ids, uint64_t k, uint64_t start_pos, qe_kv* kv,
              float* logits_out);
/* qe_verify with each row's greedy token taken on the device (the decode step's argmax rule):
 * tokens_out[i] = the token after ids[i]. */
int qe_verify_greedy(qe_model* model, const uint32_t* ids, uint64_t k, uint64_t start_pos, qe_kv* kv,
                     uint32_t* tokens_out);

/* ---- speculative greedy decode by prompt lookup (no reference counterpart: README.md:109-111
 *      names it as the next step). Same contract and same greedy tokens as qe_decode(first,
 *      start_pos, steps): each pass drafts up to k_max tokens that followed an earlier
 *      occurrence of the history's last g tokens (g = ngram .. 1; history = context[0..n_context)
 *      + first + the tokens emitted so far; the most recent occurrence with k_max followers, else
 *      the earliest) and checks them with one verify pass; drafts are
 *      accepted while they equal the greedy token of the row before, and that pass adds one
 *      greedy token of its own. With no draft a pass is one decode step. on_token gets every
 *      token in order. k_max 1..63, ngram >= 1. ---- */
typedef struct {
  uint64_t passes;        /* verify passes */
  uint64_t drafted;       /* draft tokens checked */
  uint64_t accepted;      /* draft tokens accepted */
  uint64_t single_steps;  /* decode steps taken when no draft was found */
  uint64_t plain_steps;   /* decode steps taken in plain blocks while drafting did not pay */
} qe_lookup_stats;
/* Adaptive (on unless QE_LOOKUP_ADAPTIVE=0 when the model was loaded): the host times the passes
 * as they run; once they average under 2 tokens each it also times one block of 16 pipelined
 * decode steps, and while the passes emit fewer tokens per second than those steps, it decodes
 * plain blocks of 16 steps with one pass after each (plain_steps). The tokens do not change. */
int qe_decode_lookup(qe_model* model, const uint32_t* context, uint64_t n_context, uint32_t first, uint64_t start_pos,
                     uint64_t steps, qe_kv* kv, uint32_t k_max, uint32_t ngram, qe_on_token on_token, void* user,
                     qe_lookup_stats* stats);
/* A draft source: writes up to k_max tokens that are to follow history[0..n) (context, first and
 * the tokens emitted so far) to draft_out and returns their count (0: no draft), or
 * QE_DRAFT_ERROR when it fails: the decode then stops before another pass and returns QE_ERR_ARG,
 * with the tokens emitted so far delivered and the cache valid up to the next position. */
#define QE_DRAFT_ERROR 0xFFFFFFFFu
typedef uint32_t (*qe_draft_fn)(void* user, const uint32_t* history, uint64_t n, uint32_t k_max, uint32_t* draft_out);
/* qe_decode_lookup with the drafts of `draft` (a draft model, another lookup rule, ...) instead
 * of prompt lookup, and the adaptive rule on when adaptive != 0. No reference counterpart. */
int qe_decode_drafted(qe_model* model, const uint32_t* context, uint64_t n_context, uint32_t first, uint64_t start_pos,
                      uint64_t steps, qe_kv* kv, uint32_t k_max, qe_draft_fn draft, void* draft_user, int adaptive,
                      qe_on_token on_token, void* user, qe_lookup_stats* stats);
/* The draft rule alone (host code, no device): writes the draft qe_decode_lookup would check
 * after history[0..n) (at most k_max tokens) to draft_out and returns its length. */
uint64_t qe_lookup_draft(const uint32_t* history, uint64_t n, uint32_t ngram, uint32_t k_max, uint32_t* draft_out);

/* ---- per-stage kernel timing: runs `token` at `pos` like qe_forward, then times each stage
 *      of the step (qkv, attention, o_proj, gate_up, down, lm_head, argmax) as a graph of that
 *      stage's launches only (28 per-layer launches, or one; past 1024 positions o_proj is 56:
 *      the attention merge and o_proj), replayed 8 times between two HIP
 *      events, each stage from the step state of `pos`. Writes, per stage, the mean duration of
 *      one launch in microseconds to us_out, the launches per decode step to launches_out
 *      (nullable) and the stage name (a static string) to names_out (nullable); *n_out = stages
 *      written. The stage "qkv+attention" times each layer's q|k|v and attention launches together
 *      (2 per layer), so that the attention's time behind its producer is that minus the "qkv"
 *      stage's; the stages "qkv+attention+o_proj", ... up to
 *      "qkv+attention+o_proj+gate_up+down+lm_head" time the step's prefixes the same way, so that
 *      differences of consecutive prefixes (duration x launches) are the stages' costs inside the
 *      step (the argmax, the last launch, is timed alone only: its replays advance the step
 *      state). A cache of fewer than 9 positions skips the argmax stage (its replays advance the
 *      token ring). With two launches per layer (qe_model_fused_layers() == 1) the stages are
 *      attn_block, mlp_block, final_reduce, lm_head and argmax, their prefixes and "step" (the
 *      whole step's graph); then "in_step:attn_block" and "in_step:mlp_block", each layer
 *      launch's share of the whole step (its first workgroup's start to the next layer launch's
 *      first start, from per-workgroup clock stamps of a compilation of the same kernels that
 *      writes them; launches_out counts the launches with a successor), and "in_exec:attn_block",
 *      "in_exec:mlp_block", first start to last workgroup exit. Afterwards the step is run once
 *      more, so the cache holds what qe_forward(token, pos) leaves; a kernel error raised by any
 *      replay is returned as QE_ERR_KERNEL. No reference counterpart: the reference timed kernels
 *      by removing them by hand (README.md:64-71). ---- */
int qe_profile_step(qe_model* model, uint32_t token, uint64_t pos, qe_kv* kv, float* us_out,
                    uint32_t* launches_out, const char** names_out, uint32_t max_stages, uint32_t* n_out);

/* ---- synthetic inputs (the reference loads a real checkpoint; this build writes a seeded
 *      random-init one with the same tensor names, shapes and file format) ---- */
/* Writes <dir>/model.safetensors and <dir>/config.json: every matrix bf16 ~ N(0, 0.02) from
 * `seed`, norm gains 1.0, lm_head.weight a byte copy of model.embed_tokens.weight. */
int qe_write_random_checkpoint(const char* dir, uint64_t seed, const qe_config* cfg);
/* n token ids uniform in [0, vocab) from `seed` */
void qe_random_prompt(uint64_t seed, uint64_t n, uint32_t vocab, uint32_t* out);

/* ---- isolated device ops on caller-owned device memory (HIP device pointers; stream may be
 *      NULL for the default stream). For the isolated benchmarks and kernel parity tests. ---- */
/* out[r] = sum_c bf16(w[r*cols + c]) * x[c], f32 accumulate; matvec_bf16,
 * inference.metal:143-186 / cpu_inference.rs:225-257. cols % 8 == 0, w 16-byte aligned. */
int qe_op_matvec_bf16(const void* w, const float* x, float* out, uint64_t rows, uint64_t cols,
                      void* stream);
/* c[i][j] = sum_k a[i][k] bf16(w[j][k]): the chunked prefill's GEMM (a f32 [m][k] split into two
 * bf16 halves, w bf16 [n][k], f32 accumulate on the matrix cores). n even, k % 32 == 0,
 * a and w 16-byte aligned. No reference counterpart (the reference has no batched path). */
int qe_op_gemm_bf16(const float* a, const void* w, float* c, uint64_t m, uint64_t n, uint64_t k,
                    void* stream);
/* One decode step of GQA attention (cpu_inference.rs:144-162, inference.metal:234-296) for
 * head_dim 128: q [n_heads*128] (post q-norm and RoPE), k/v caches laid out
 * [n_kv_heads][kv_stride][128] f32, attending positions 0..n_pos-1; out [n_heads*128].
 * The positions are split into n_splits runs (1..128; 0 picks runs of 64 positions), each
 * attended by one workgroup per KV head, and a second kernel merges the runs' partial softmax
 * sums; with n_splits = 0, up to 256 positions and 1 or 2 q heads per KV head, one kernel does
 * both unless out overlaps q, k or v (it may, in either form: they are read before it is
 * written). `work` (partials, overwritten by every call) must hold qe_op_attention_work_bytes(...)
 * bytes of device memory. */
uint64_t qe_op_attention_work_bytes(uint64_t n_heads, uint64_t n_kv_heads, uint64_t n_pos);
int qe_op_attention(const float* q, const float* k, const float* v, float* out, uint64_t n_pos,
                    uint64_t kv_stride, uint64_t n_heads, uint64_t n_kv_heads, uint32_t n_splits,
                    void* work, void* stream);
/* qe_op_attention with no work buffer and no allocation: the partial sums go to a 1 MiB array in
 * device memory that the library holds on each GPU it runs on until the process ends. No
 * counterpart in the reference: it is for callers that cannot allocate device memory (code under
 * HIP graph capture, serving loops that forbid hipMalloc). Same arguments and results as
 * qe_op_attention; calls with n_heads x runs above 2048 (runs = n_splits, or n_pos / 64 rounded
 * up, at most 128) are refused with QE_ERR_ARG. Every call on one GPU shares that GPU's array, so
 * calls that overlap on one GPU (two streams or two threads) race. The first call on each device
 * looks up the array's device address (hipGetSymbolAddress, which may load the library's device
 * code): make it outside stream capture; later calls may be captured into a graph. */
int qe_op_attention_static(const float* q, const float* k, const float* v, float* out, uint64_t n_pos,
                           uint64_t kv_stride, uint64_t n_heads, uint64_t n_kv_heads, uint32_t n_splits,
                           void* stream);
/* Greedy token of each of `rows` logit rows of n floats (device memory, row-major): the argmax
 * of main.rs:37-42 -- the first maximum wins (lowest index on ties, -0.0 ties +0.0), NaN entries
 * never win, a NaN at index 0 gives 0, and a row with nothing above -inf gives 0. tokens_out:
 * `rows` uint32 in device memory. The verify pass's device argmax (qe_verify_greedy) runs this
 * kernel. */
int qe_op_argmax(const float* logits, uint64_t rows, uint64_t n, uint32_t* tokens_out, void* stream);
/* Streaming read of n floats (n % 4 == 0): the read_sum kernel of tests/read_bandwidth.rs:16-54,
 * writing one partial sum per block to partial[grid]. grid == 0 picks a default. */
int qe_op_read_sum(const float* src, uint64_t n, float* partial, uint32_t grid, void* stream);
/* The same sum with non-temporal loads (not allocated in the MALL), block b reading the contiguous
 * quarter-float4 range [n/4 b / grid, n/4 (b + 1) / grid): on gfx950 this streaming form reads
 * faster than the strided one, so the read ceiling is the better of the two. It replaces nothing
 * in the reference, whose read_bandwidth.rs kernel has one form (tests/read_bandwidth.rs:16-54). */
int qe_op_read_sum_nt(const float* src, uint64_t n, float* partial, uint32_t grid, void* stream);

/* ---- paged K/V cache for several sequences, and the attention that reads it: operators on
 *      caller-owned device memory, for one layer. No reference counterpart: its cache is one
 *      buffer per layer and sequence (metal_inference.rs:115-138). ----
 * Pages hold K and V of page_size positions each (a power of two, 16..65536), head_dim 128, as bf16
 * or e4m3 (QE_KV_BF16, QE_KV_FP8):
 *   k [n_pages][n_kv_heads][page_size][128]
 *   v [n_pages][n_kv_heads][page_size / 16][128][16]: each 16 positions transposed, the form in
 *     which the matrix cores take V
 * and, with QE_KV_FP8, one exponent byte e per position and KV head in k_exp and v_exp
 * [n_pages][n_kv_heads][page_size]: the row's values are the stored ones times 2^(e - 127), e from
 * 1 to 254.
 * The plan of a call is device memory too, read when the call runs: row s of `table` names the
 * pages of sequence s in order, lens[s] is its length with the call's new tokens, and the packed
 * rows starts[s] .. starts[s + 1] are its new tokens, the last of them at position lens[s] - 1
 * (starts has n_seqs + 1 entries and does not decrease). A table entry outside 0 .. n_pages - 1, or
 * a position past the table, means that the page is not there. Packed rows that belong to no
 * sequence are left as they were. Pages may be shared by sequences that only read them. */
typedef struct qe_pages {
  void* k;               /* 16-byte aligned, as v and the exponents */
  void* v;
  uint8_t* k_exp;        /* QE_KV_FP8 only */
  uint8_t* v_exp;
  const int32_t* table;  /* [n_seqs][table_stride] */
  const int32_t* lens;   /* [n_seqs] */
  const int32_t* starts; /* [n_seqs + 1] */
  uint64_t n_pages;      /* below 2^31 */
  uint64_t page_size;
  uint64_t n_kv_heads;   /* 1..1024 */
  uint64_t n_seqs;       /* 1..65536 */
  uint64_t table_stride; /* table_stride * page_size below 2^31 */
  int kv_dtype;
} qe_pages;
/* Bytes of k, and of v (0 for another kv_dtype). */
uint64_t qe_page_bytes(uint64_t n_pages, uint64_t page_size, uint64_t n_kv_heads, int kv_dtype);
/* Writes the new tokens' K and V rows into their pages: k, v [n_rows][n_kv_heads][128] of dtype
 * QE_KV_F32 or QE_KV_BF16, rows row_stride elements apart, 16-byte aligned. bf16 pages take the
 * nearest value. e4m3 pages: the exponent is the smallest for which the row's largest finite
 * magnitude is at most 448 of its scale, the values are the nearest (ties to even), and infinities
 * and NaN become NaN. A position whose page is not there is not written. Two rows for one position
 * of one page: either may win. n_rows, rounded up to a multiple of 16, times n_kv_heads must be below
 * 2^28; n_rows = 0 does nothing. */
int qe_op_page_append(const qe_pages* pages, const void* k, const void* v, uint64_t n_rows, uint64_t row_stride,
                      int dtype, void* stream);
/* The same rows out of the pages (arguments as qe_op_page_append; k and v are written): zeros where
 * a page is not there. */
int qe_op_page_read(const qe_pages* pages, void* k, void* v, uint64_t n_rows, uint64_t row_stride, int dtype,
                    void* stream);
/* Causal GQA attention of the new tokens over the pages (their own K and V appended before):
 * out[t][h] = softmax over j <= position of t of (q[t][h] . k[j] / sqrt(128)), times v[j], over the
 * positions whose page is there; zeros for a row that has none. q and out are [n_rows][n_heads][128]
 * of `dtype` (QE_KV_F32 or QE_KV_BF16), rows q_stride and out_stride elements apart, 16-byte
 * aligned; an out that overlaps q or the pages is refused (rows of out may lie between those of q).
 * n_heads is a multiple of n_kv_heads. Softmax and sums are f32; f32 rows keep f32's precision, bf16
 * rows take the softmax weights (e4m3 pages: times V's scale) rounded to bf16, each by at most 2^-8 of
 * itself. Weights are up to 2^8 before the division by their sum, so sums over V of magnitudes up to
 * 2^88 stay finite at any length; far larger ones may become infinite. A position that a row does not
 * attend has no part in it, whatever K and V hold there; infinities and NaN where it does attend may
 * make it either.
 * max_new: the most new tokens any sequence has (0: not known). It chooses how the work is cut up;
 * the results are right for any value, but the tiles are as large as the longest sequence wants: a call
 * of a long chunk beside many sequences of one token takes longer than one call for each kind, and one
 * with 0 may take longer than with the right value. `work` is scratch memory of the call, overwritten by every
 * call: work_bytes at least what qe_op_page_attention_work_bytes gives for the same values. Calls
 * that may overlap need one each. n_rows = 0 does nothing. */
uint64_t qe_op_page_attention_work_bytes(uint64_t n_heads, uint64_t n_kv_heads, uint64_t max_new);
int qe_op_page_attention(const qe_pages* pages, const void* q, void* out, uint64_t n_rows, uint64_t n_heads,
                         uint64_t q_stride, uint64_t out_stride, uint64_t max_new, int dtype, void* work,
                         uint64_t work_bytes, void* stream);
/* The same for trees of drafted tokens: the new tokens of a sequence are the nodes of a tree (or of
 * several), at most QE_TREE_NODES of them, appended like any new tokens: node i at position
 * lens[s] - new + i. parents [n_rows] (int32): which of its sequence's rows a node's parent is, an
 * earlier one (0 .. i - 1); any other value: it has none. A node attends the positions before the new
 * tokens, its ancestors and itself; what the others hold has no part in it. A row behind its sequence's
 * first QE_TREE_NODES is zeros. max_new: at most QE_TREE_NODES; work_bytes and all else as
 * qe_op_page_attention, and out and work must not overlap parents. */
#define QE_TREE_NODES 64
int qe_op_page_tree_attention(const qe_pages* pages, const int32_t* parents, const void* q, void* out, uint64_t n_rows,
                              uint64_t n_heads, uint64_t q_stride, uint64_t out_stride, uint64_t max_new, int dtype,
                              void* work, uint64_t work_bytes, void* stream);

/* ---- a cache of bounded size: which positions get attention, which to keep, and the move of kept rows
 *      to the front. No reference counterpart. ----
 * mass [n_seqs][n_kv_heads][mass_stride] (f32) belongs to the sequences of a plan: entry j of a sequence
 * and KV head is the softmax weight that position j got so far. */
/* Adds to mass the weights that the new tokens give: mass[s][h][j] += sum over rows t of sequence s and q
 * heads g of KV head h of the softmax weight of position j in (t, g), as qe_op_page_attention weighs
 * them (causal; a position whose page is not there gets nothing). Arguments as there: the rows are the
 * last tokens of their sequences, so a call may also take only the last few of a prompt. mass_stride is
 * at least table_stride * page_size. Weights and sums are f32, of rows of either type; the sums are the
 * same every time. A row with a score that is not finite may make any position it attends NaN. mass
 * must not overlap q, the pages or work. n_rows * n_heads is below 2^28, and n_seqs * n_kv_heads times the
 * positions of a table's row / 256 below 2^24. max_new as there; with more new tokens than it says a call may take
 * much longer, never give another result than its sums' rounding. work is scratch of the call, of the size for the same
 * values (positions: table_stride * page_size); calls that may overlap need one each. */
uint64_t qe_op_page_weigh_work_bytes(uint64_t n_rows, uint64_t n_heads, uint64_t n_kv_heads, uint64_t n_seqs,
                                     uint64_t positions, uint64_t max_new);
int qe_op_page_weigh(const qe_pages* pages, const void* q, uint64_t n_rows, uint64_t n_heads, uint64_t q_stride,
                     uint64_t max_new, int dtype, float* mass, uint64_t mass_stride, void* work, uint64_t work_bytes,
                     void* stream);
/* Picks the positions that each KV head of a sequence keeps, by mass: count[s] = min(lens[s], keep) of
 * 0 .. lens[s] - 1 (lens below 0 counts as 0, above mass_stride as mass_stride), the first `sinks` and the
 * last `recent` of them always (sinks + recent at most keep), the others by the largest mass, the lowest
 * position on ties; NaN counts as the smallest, -0 as 0. kept [n_seqs][n_kv_heads][kept_stride]: the
 * positions, ascending, then -1 up to `keep` (1 .. kept_stride; the rest of a row is left as it was).
 * mass_stride and kept_stride below 2^31, n_seqs * n_kv_heads below 2^22. Outputs must not overlap the inputs. */
int qe_op_page_keep(const float* mass, uint64_t mass_stride, const int32_t* lens, uint64_t n_seqs, uint64_t n_kv_heads,
                    uint64_t keep, uint64_t sinks, uint64_t recent, int32_t* kept, uint64_t kept_stride,
                    int32_t* count, void* stream);
/* Moves rows of the pages to the front, in place, K, V and their exponents: position first[s] + i of
 * sequence s takes the row at first[s] + src[s][h][i], for i < count[s]. src [n_seqs][src_heads][src_stride]
 * (int32): src_heads is 1 (all KV heads alike) or n_kv_heads; a row of it ascends, with src[i] >= i. So
 * qe_op_page_keep's positions pack what was kept (first NULL: 0), and qe_op_verify_tree's path puts the
 * accepted nodes one after another (first: lens before the nodes). mass (nullable) moves along, and is
 * 0 from first[s] + count[s] to lens[s]; lens itself is the caller's to change. A row whose source or
 * destination is not there (a page that is not, a position past the table or, for mass, mass_stride) is
 * left as it was; src that does not ascend or has src[i] < i leaves some of the rows moved undefined, and no
 * others. count above src_stride counts as src_stride. A page that two sequences share is moved by both:
 * not for shared pages. src_stride and mass_stride are below 2^31, n_seqs * n_kv_heads below 2^19,
 * the rows of all pages (n_pages * n_kv_heads * page_size) below 2^32 - 1. */
int qe_op_page_move(const qe_pages* pages, const int32_t* src, uint64_t src_heads, uint64_t src_stride,
                    const int32_t* count, const int32_t* first, float* mass, uint64_t mass_stride, void* stream);

/* ---- drafted tokens against the target's probabilities, from given random numbers: the sampled
 *      form of qe_verify_greedy's rule, on device memory. No reference counterpart. ----
 * Rows starts[s] .. starts[s + 1] of the logits [n_rows][vocab] (f32, rows row_stride apart) are
 * sequence s's: one per draft and one for the token after the last. Row r's target is
 * p = softmax(logits / temperature[s]); drafts[r] is its drafted token (the last row of a sequence
 * has none) and draft_probs[r] (rows probs_stride apart) what it was drawn from. The drafts are
 * accepted in order while accept[r] * draft_probs[r][d] < p[d]. The first row that does not accept
 * draws its token from max(p - draft_probs[r], 0); the last row draws from p. A draw takes the
 * smallest token whose running sum of weights is above sample[s] times their sum. accept [n_rows]
 * and sample [n_seqs] are numbers in [0, 1). With draft_probs NULL each draft was certain
 * (probability 1), as a lookup's are. temperature NULL is 1; one that is not above 0 is greedy: all
 * of p on the first largest logit. NaN logits count as -inf, infinite ones share p; a row with
 * nothing above -inf gives token 0. Draft probabilities that are not above 0 count as 0, and where
 * nothing is left of p - q the draw is from p. A draft that is not below vocab is not accepted.
 * tokens_out [n_rows]: each sequence's accepted drafts, then the drawn token, then 0xFFFFFFFF;
 * count_out [n_seqs]: how many tokens that is (0 for a sequence without rows); logprobs_out
 * [n_rows] (nullable): log p of each, 0 behind them. Rows that belong to no sequence are left as
 * they were. Sums are f64. vocab 1..2^20, n_seqs 1..65535. `work` as qe_op_page_attention's. */
uint64_t qe_op_verify_drafts_work_bytes(uint64_t n_rows, uint64_t n_seqs, uint64_t vocab);
int qe_op_verify_drafts(const float* logits, uint64_t n_rows, uint64_t vocab, uint64_t row_stride,
                        const int32_t* starts, uint64_t n_seqs, const uint32_t* drafts, const float* draft_probs,
                        uint64_t probs_stride, const float* accept, const float* sample, const float* temperature,
                        uint32_t* tokens_out, uint32_t* count_out, float* logprobs_out, void* work,
                        uint64_t work_bytes, void* stream);


/* The same for a tree of drafts. Rows starts[s] .. starts[s + 1] are the nodes of sequence s's tree, row
 * starts[s] its root: the last token that is certain. The logits of a row are the target's after the tokens
 * from the root to it; nodes[r] is its own token (the root's is not read) and parents[r] says which of
 * the sequence's rows it follows, as in qe_op_page_tree_attention; a node without a parent other than
 * the root, and a row behind the first QE_TREE_NODES, is never reached. From the root on: with p = softmax(logits
 * of the node / temperature[s]), the node's children are tried in the order of their rows; child c is accepted
 * while accept[c] * (1 - sum of the p of those tried before) < p[nodes[c]], a token that was tried before
 * having no p left. The walk goes on from the first accepted child. Where none is, or max_depth drafts
 * (0: no bound; large trees are checked faster with one) have been accepted, the last token is drawn from p
 * without the tokens tried (of a node at max_depth none are) by sample[s]. What is emitted follows the target's distribution whatever the tree is.
 * accept [n_rows] and sample [n_seqs] are numbers in [0, 1). Logits, temperature, draws, logprobs_out and work
 * as in qe_op_verify_drafts; tokens_out [n_rows]: the accepted nodes' tokens, then the drawn one, then
 * 0xFFFFFFFF; path_out [n_seqs][QE_TREE_NODES] (int32): 0 for the root, the accepted nodes' rows counted from
 * starts[s], then -1; count_out [n_seqs]: how many tokens, and rows on the path, that is (0 for a sequence
 * without rows). So path_out and count_out are the src and count of qe_op_page_move. */
uint64_t qe_op_verify_tree_work_bytes(uint64_t n_rows, uint64_t n_seqs, uint64_t vocab);
int qe_op_verify_tree(const float* logits, uint64_t n_rows, uint64_t vocab, uint64_t row_stride, const int32_t* starts,
                      uint64_t n_seqs, const int32_t* parents, const uint32_t* nodes, const float* accept,
                      const float* sample, const float* temperature, uint64_t max_depth, uint32_t* tokens_out,
                      int32_t* path_out, uint32_t* count_out, float* logprobs_out, void* work, uint64_t work_bytes,
                      void* stream);

#ifdef __cplusplus
}
#endif
#endif
