/*
 * flashtrie_b200 - C ABI of the B200 trie-constrained beam search (TBS) engine.
 *
 * This is the drop-in boundary for the reference FlashTrie TBS path: every
 * entry point below replaces one call the reference's pybind11 module
 * `flashtrie` (tools/bindings.cpp) makes into `marisa::Trie`
 * (include/marisa/trie.h).  Plain pointers and sizes only; no exceptions
 * cross the ABI.  Every function returns FT_OK (0) or a negative FT_ERR_*
 * code; ft_last_error() gives the message of the calling thread's last
 * failure.
 *
 * Memory layout conventions:
 *   - a request has L decoding positions (L = len(beams)) and K proposals per
 *     position; rows are stored row-major: topk_id[t*K + j], topk_logp[t*K + j];
 *   - results are ascending by logp_norm, like the reference output
 *     (lib/marisa/grimoire/trie/tbs-kernels.cu:415-421).
 */
#ifndef FLASHTRIE_B200_H_
#define FLASHTRIE_B200_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes.  -1..-10 mirror marisa_error_code (include/marisa/base.h:79-91). */
#define FT_OK 0
#define FT_ERR_STATE (-1)    /* MARISA_STATE_ERROR: no trie, no workspace, ...   */
#define FT_ERR_NULL (-2)     /* MARISA_NULL_ERROR                                */
#define FT_ERR_BOUND (-3)    /* MARISA_BOUND_ERROR                               */
#define FT_ERR_RANGE (-4)    /* MARISA_RANGE_ERROR                               */
#define FT_ERR_CODE (-5)     /* MARISA_CODE_ERROR: bad config flags              */
#define FT_ERR_SIZE (-7)     /* MARISA_SIZE_ERROR: trie exceeds format limits    */
#define FT_ERR_MEMORY (-8)   /* MARISA_MEMORY_ERROR / device allocation failed   */
#define FT_ERR_IO (-9)       /* MARISA_IO_ERROR                                  */
#define FT_ERR_FORMAT (-10)  /* MARISA_FORMAT_ERROR                              */
#define FT_ERR_INVALID_ARG (-20) /* request violates the workspace limits        */
#define FT_ERR_CUDA (-21)        /* a CUDA runtime call failed                   */
#define FT_ERR_DEVICE (-22)      /* the search kernel reported a bad trie access */

typedef struct ft_trie ft_trie;

typedef struct {
  uint64_t num_keys;   /* Trie::num_keys   (include/marisa/trie.h:51)  */
  uint64_t num_nodes;  /* Trie::num_nodes  (include/marisa/trie.h:52)  */
  uint64_t num_tries;  /* Trie::num_tries  (include/marisa/trie.h:50)  */
  uint64_t total_size; /* Trie::total_size (include/marisa/trie.h:59)  */
  uint64_t io_size;    /* Trie::io_size    (include/marisa/trie.h:60)  */
  uint32_t tail_mode;  /* Trie::tail_mode  (include/marisa/trie.h:54)  */
  uint32_t node_order; /* Trie::node_order (include/marisa/trie.h:55)  */
} ft_trie_info;

/* One request, host memory (TbsInput inputs, include/marisa/tbs_input.h:7-12). */
typedef struct {
  uint32_t num_outpos;        /* L = len(beams)                       */
  uint32_t topk;              /* K, proposals per position            */
  const uint32_t *beams;      /* [L] beam width per position           */
  const uint32_t *topk_id;    /* [L*K] token ids                       */
  const float *topk_logp;     /* [L*K] token log-probabilities         */
} ft_request;

/* One result, host memory (TbsInput outputs, include/marisa/tbs_input.h:13-25).
 * The caller provides capacity >= beams[L-1] and stride >= L. */
typedef struct {
  uint32_t capacity;          /* in: beams the arrays can hold               */
  uint32_t stride;            /* in: token slots per beam                    */
  uint32_t num_beams;         /* out                                         */
  uint32_t reserved;
  double *logp_norm;          /* out: [capacity], ascending                  */
  uint32_t *lengths;          /* out: [capacity]                             */
  uint32_t *tokens;           /* out: [capacity*stride], beam i at i*stride  */
  double phase_ms[5];         /* out: expansion, validation, selection,
                                 overhead, kernel (tbs_input.h:19-25)        */
  uint32_t *key_ids;          /* out, optional ([capacity], NULL: not written):
                                 the key id of each beam, as LoudsTrie::lookup
                                 reports it (louds-trie.cc:56-72; no
                                 counterpart in the reference's TbsInput)    */
} ft_result;

/* Search parameters shared by a batch (tools/bindings.cpp:71-78). */
typedef struct {
  float token_logp_threshold;
  float reserved;
  double sent_logp_threshold;
  double length_norm;
  int32_t early_exit;
  int32_t reserved2;
} ft_search_params;

/* Last error message of the calling thread ("" if none). */
const char *ft_last_error(void);

/* marisa::Trie::Trie() (include/marisa/trie.h:21), bound at tools/bindings.cpp:28 */
int ft_trie_create(ft_trie **out);
/* marisa::Trie::~Trie(); frees host and device state */
void ft_trie_destroy(ft_trie *trie);

/* marisa::Trie::load (include/marisa/trie.h:29), bound at tools/bindings.cpp:29 */
int ft_trie_load(ft_trie *trie, const char *path);
/* marisa::Trie::mmap (include/marisa/trie.h:26), bound at tools/bindings.cpp:30 */
int ft_trie_mmap(ft_trie *trie, const char *path);
/* build_from_list (tools/bindings.cpp:10-22): keys as a flat token array plus
 * num_rows+1 offsets; flags 1 | TEXT_TAIL | LABEL_ORDER | NORMAL_CACHE */
int ft_trie_build(ft_trie *trie, const uint32_t *tokens, const uint64_t *offsets, uint64_t num_rows);
/* marisa::Trie::save (include/marisa/trie.h:32), bound at tools/bindings.cpp:36 */
int ft_trie_save(const ft_trie *trie, const char *path);
/* marisa::Trie::clear (include/marisa/trie.h:62), bound at tools/bindings.cpp:37 */
int ft_trie_clear(ft_trie *trie);
/* num_keys / num_nodes / num_tries / total_size / io_size
 * (tools/bindings.cpp:32-35) */
int ft_trie_get_info(const ft_trie *trie, ft_trie_info *out);

/* marisa::Trie::init_tbs_gpu (include/marisa/trie.h:40-44), bound at
 * tools/bindings.cpp:38-43.  Uploads the trie to the current CUDA device and
 * sizes the search workspace. */
int ft_trie_init_tbs_gpu(ft_trie *trie, uint64_t max_batch_size, uint64_t max_num_topk,
                         uint64_t max_num_outpos, uint64_t max_num_out_beams,
                         uint64_t max_num_out_tokens, uint64_t max_num_inter_beams,
                         uint64_t radix_topk_threshold);
/* marisa::Trie::get_max_batch_size (include/marisa/trie.h:45) */
int ft_trie_get_max_batch_size(const ft_trie *trie, uint64_t *out);

/* marisa::Trie::tbs_gpu_batched (include/marisa/trie.h:48), bound as
 * bs_tbs_gpu at tools/bindings.cpp:71-119, and marisa::Trie::tbs_gpu
 * (trie.h:47) for n == 1.  Host buffers in and out; copies, kernel and
 * synchronisation happen inside the call. */
int ft_tbs_batch(ft_trie *trie, const ft_request *requests, uint32_t n,
                 const ft_search_params *params, ft_result *results);

/*
 * Device-resident batch (no counterpart in the reference, which always stages
 * host buffers): the same search on inputs already in device memory, written
 * to device outputs, on a caller stream.  Layout of the inputs for n
 * requests with a common L and K:
 *   beams     u32 [n][L]
 *   topk_id   u32 [n][L][K]
 *   topk_logp f32 [n][L][K]
 * Every pointer of a non-empty batch except out_key must be set (the rows
 * only when K > 0); a NULL one is refused with FT_ERR_NULL before any launch.
 * Outputs, per request i, with cap = max final beam and stride = L:
 *   out_count u32 [n]            number of beams
 *   out_lpn   f64 [n][cap]       ascending logp_norm
 *   out_len   u32 [n][cap]
 *   out_tok   u32 [n][cap][L]
 *   out_key   u32 [n][cap]       key ids (optional, NULL: not written)
 * `stream` is a cudaStream_t (0 = default stream).  The call returns after
 * enqueueing; completion is observed with stream synchronisation.
 */
typedef struct {
  uint32_t n;
  uint32_t num_outpos;
  uint32_t topk;
  uint32_t out_capacity;
  const uint32_t *beams;
  const uint32_t *topk_id;
  const float *topk_logp;
  uint32_t *out_count;
  double *out_lpn;
  uint32_t *out_len;
  uint32_t *out_tok;
  uint32_t *out_key;
} ft_device_batch;

int ft_tbs_batch_device(ft_trie *trie, const ft_device_batch *batch,
                        const ft_search_params *params, void *stream);

/*
 * Replaces LoudsTrie::lookup (lib/marisa/grimoire/trie/louds-trie.cc:56-72)
 * for a batch, on the device: key i is tokens[offsets[i] .. offsets[i+1]) and
 * out_ids[i] receives its key id (the id ft_result.key_ids reports), or
 * 0xFFFFFFFF when it is not a key of the trie.  tokens (total_tokens entries),
 * offsets (n + 1 entries) and out_ids (n entries) are device pointers; the
 * lookup runs on `stream` and the call returns without waiting.  Requires
 * ft_trie_init_tbs_gpu.  Offsets that decrease or pass total_tokens give
 * 0xFFFFFFFF for that key and set a bit of the device status word.
 */
int ft_lookup_batch_device(ft_trie *trie, uint32_t n, const uint32_t *tokens, const uint64_t *offsets,
                           uint64_t total_tokens, uint32_t *out_ids, void *stream);

/*
 * Replaces LoudsTrie::reverse_lookup (lib/marisa/grimoire/trie/louds-trie.cc:179-210)
 * for a batch, on the device: out_len[i] receives the length of the key whose
 * id is ids[i] (0xFFFFFFFF when ids[i] is not a key id), and its tokens go to
 * out_tokens[i * max_len ...] when that length is at most max_len.  ids (n),
 * out_tokens (n * max_len) and out_len (n) are device pointers; the lookup
 * runs on `stream` and the call returns without waiting.  Requires
 * ft_trie_init_tbs_gpu; the first call derives every node's parent (4 bytes
 * per node, freed with the workspace) and waits for that once.
 */
int ft_reverse_lookup_batch_device(ft_trie *trie, uint32_t n, const uint32_t *ids, uint32_t max_len,
                                   uint32_t *out_tokens, uint32_t *out_len, void *stream);

/* Status word of the device-resident searches and lookups since the last call
 * (0 = clean; the word is cleared by reading it); non-zero bits name the
 * checks that failed inside the kernel. */
int ft_trie_device_status(ft_trie *trie, uint32_t *status);
/* The device address of that word, for calls on the same device that report
 * into it (ft_adapter_logits_checked_device).  It is the trie's until its GPU
 * workspace is made anew or the trie destroyed. */
int ft_trie_status_word(ft_trie *trie, uint32_t **word);

/*
 * No counterpart in the reference.  The same search as ft_tbs_batch_device,
 * for callers that cannot allocate device memory while they search: code whose
 * host framework owns every device allocation, or request threads that must
 * not stall on cudaMalloc/cudaFree.  It allocates nothing; its scratch is a
 * fixed 8 MiB array in the library, which every GPU that loads the library
 * keeps until exit.  The trie must already be on the device
 * (ft_trie_init_tbs_gpu); the caller passes device inputs and outputs as for
 * ft_tbs_batch_device, with every beam width at most out_capacity.  Batches
 * whose scratch would exceed 8 MiB are rejected with FT_ERR_INVALID_ARG.
 * The first call on a device looks up the array's address; make it before any
 * stream capture.  Calls are serialised per device; each reads the kernel's
 * status word back on `stream` and synchronises `stream` before it returns,
 * so no call can be made inside a stream capture.  All calls share the array, so searches whose GPU work overlapped would race.
 */
int ft_tbs_batch_device_noalloc(ft_trie *trie, const ft_device_batch *batch,
                                const ft_search_params *params, void *stream);

/*
 * Model-side operators around the search (no counterpart in the reference,
 * whose callers bring topk_id / topk_logp with them): the vocabulary
 * projection that gives the logits, the proposals taken from them, and the
 * scores and preference loss of the sequences that the search found.
 *
 * They belong to no trie.  Every pointer is a device pointer on the current
 * CUDA device, arrays are dense and row-major; `stream` is a cudaStream_t of
 * that device.  The calls only enqueue and may be captured into a CUDA graph.
 * They allocate nothing: the caller passes `workspace`, 256-byte aligned, of
 * at least the bytes the matching *_workspace call reports, which no other
 * call may use until this one's work has finished.  Its contents need no
 * initialisation.
 */
#define FT_DTYPE_F32 0
#define FT_DTYPE_BF16 1
#define FT_DTYPE_F16 2

/*
 * Logits of n requests with num_outpos positions each:
 *   out[i][l][v] = sum_d hidden[i][l][d] weight[v][d]
 *                + scale[a] sum_r (sum_d hidden[i][l][d] lora_a[a][r][d]) lora_b[a][v][r]
 * with a = adapter_ids[i].  a = -1: the shared projection alone; any other id
 * outside [0, num_adapters) makes the request's logits NaN.  hidden, weight,
 * lora_a and lora_b are dtype (bf16 or f16), out is out_dtype (the same type,
 * or f32); all five start on 16-byte boundaries.  dim and rank are multiples
 * of 8, rank at most 256.  scale * (hidden lora_a) may have any size that f32
 * holds; 2^-17 of it is lost at most (2^-26 with bf16 operands and f32 logits),
 * with f16 operands 2^-23, or 2^-25 absolute and 2^-17 of the token's largest.
 * An infinite one, or an infinity in lora_b, makes the logits that it enters NaN
 * or infinite.  out overlaps none of the inputs.  num_adapters = 0: adapter_ids, lora_a, lora_b and
 * scale are not read.  scale may be NULL (1 for every adapter).  At most
 * 65536 adapters.
 */
typedef struct {
  uint32_t n;
  uint32_t num_outpos;
  uint32_t vocab;
  uint32_t dim;
  uint32_t rank;
  uint32_t num_adapters;
  int32_t dtype;
  int32_t out_dtype;
  const void *hidden;          /* [n][num_outpos][dim]            */
  const void *weight;          /* [vocab][dim]                    */
  const int32_t *adapter_ids;  /* [n]                             */
  const void *lora_a;          /* [num_adapters][rank][dim]       */
  const void *lora_b;          /* [num_adapters][vocab][rank]     */
  const float *scale;          /* [num_adapters] or NULL          */
  void *out;                   /* [n][num_outpos][vocab]          */
} ft_adapter_args;

int ft_adapter_logits_workspace(const ft_adapter_args *args, uint64_t *bytes);
int ft_adapter_logits_device(const ft_adapter_args *args, void *workspace, uint64_t workspace_bytes, void *stream);
/* The same with a status word in device memory (or NULL): the kernel's waits
 * are bounded, and where one runs out it sets a bit of *status and leaves NaN in
 * the logits that it has not made.  Nothing clears the word. */
int ft_adapter_logits_checked_device(const ft_adapter_args *args, uint32_t *status, void *workspace,
                                     uint64_t workspace_bytes, void *stream);

/*
 * The search's proposals from logits: per row, log-softmax over the
 * vocabulary and its topk largest entries, equal logits in order of the token
 * id.  order 0: each row ascending by id (what the search reads without
 * sorting); 1: by descending log-probability, then id.  Entries with a logit
 * of -inf are never proposed; a row with fewer than topk others ends with
 * entries (0xFFFFFFFF, -FLT_MAX), which no search step takes, and so does,
 * from its start, a row without a distribution (a NaN or +inf among its
 * logits, or -inf alone).  topk is in [1, 8192].
 */
typedef struct {
  uint64_t rows;        /* n * num_outpos                 */
  uint32_t vocab;
  uint32_t topk;
  int32_t dtype;
  int32_t order;
  const void *logits;   /* [rows][vocab]                  */
  uint32_t *topk_id;    /* [rows][topk]                   */
  float *topk_logp;     /* [rows][topk]                   */
} ft_propose_args;

int ft_propose_workspace(const ft_propose_args *args, uint64_t *bytes);
int ft_propose_device(const ft_propose_args *args, void *workspace, uint64_t workspace_bytes, void *stream);

/*
 * Scores of candidate sequences under the logits of their request:
 *   logp[i][j] = sum over l < lengths[i][j] of log softmax(logits[i][l])[tokens[i][j][l]]
 * tokens and lengths have the layout of the search's results (out_tok,
 * out_len with out_capacity = candidates).  Length 0 gives 0; a length
 * outside [0, num_outpos] gives NaN and takes no part in gradients; tokens
 * behind a length do not matter.  A token id >= vocab counts as a logit of
 * -inf, and so does every token of a position whose logits are all -inf; such
 * a position has no gradient.  candidates is at most 8192.  `stats` receives
 * (maximum, sum of exponentials) of every row, which the gradient reads.
 */
typedef struct {
  uint32_t n;
  uint32_t num_outpos;
  uint32_t vocab;
  uint32_t candidates;
  int32_t dtype;
  int32_t reserved;
  const void *logits;       /* [n][num_outpos][vocab]             */
  const uint32_t *tokens;   /* [n][candidates][num_outpos]        */
  const int32_t *lengths;   /* [n][candidates]                    */
  float *stats;             /* [n][num_outpos][2]                 */
  float *logp;              /* [n][candidates], NULL: not written */
  void *grad_logits;        /* [n][num_outpos][vocab], gradients  */
} ft_sequence_args;

int ft_sequence_logp_workspace(const ft_sequence_args *args, uint64_t *bytes);
int ft_sequence_logp_device(const ft_sequence_args *args, void *workspace, uint64_t workspace_bytes, void *stream);
/* grad_logits = the gradient of sum_ij w[i][j] logp[i][j], with w = grad
 * ([n][candidates]), times *factor and *upstream (device scalars, each may be
 * NULL).  Reads stats as the forward call left it; grad_logits may not overlap
 * logits. */
int ft_sequence_grad_device(const ft_sequence_args *args, const float *grad, const float *factor,
                            const float *upstream, void *workspace, uint64_t workspace_bytes, void *stream);

/*
 * Preference loss on pairs of candidates of the same request:
 *   margin = beta ((logp[c] - ref_logp[c]) - (logp[r] - ref_logp[r]))
 *   loss   = sum over pairs of (1 - s) softplus(-margin) + s softplus(margin),
 * s = label_smoothing, in [0, 1]; beta is finite; with `mean`, divided by the number of pairs (at least
 * 1).  A pair with a negative index is absent: margin 0, no loss.  One with
 * an index >= candidates makes its margin and the loss NaN and has no
 * gradient.  grad receives d loss / d logp before that division and factor
 * the division, in the form that ft_sequence_grad_device takes.
 */
typedef struct {
  uint32_t pairs;           /* pairs per request                  */
  int32_t mean;
  float beta;
  float label_smoothing;
  const float *ref_logp;    /* [n][candidates]                    */
  const int32_t *chosen;    /* [n][pairs]                         */
  const int32_t *rejected;  /* [n][pairs]                         */
  float *margin;            /* [n][pairs]                         */
  float *loss;              /* [1]                                */
  float *grad;              /* [n][candidates]                    */
  float *factor;            /* [1]                                */
} ft_preference_args;

int ft_preference_loss_workspace(const ft_sequence_args *args, uint64_t *bytes);
int ft_preference_loss_device(const ft_sequence_args *args, const ft_preference_args *pref, void *workspace,
                              uint64_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* FLASHTRIE_B200_H_ */
