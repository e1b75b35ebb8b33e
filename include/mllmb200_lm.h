/*
 * mllmb200_lm.h - C ABI of the bf16 language-model engine (library lib/libmllm_b200_lm.so).
 *
 * The engine runs decoder-only models that are described layer by layer: a sequence mixer (softmax attention, latent
 * attention or retention), an optional gated feed-forward (dense or a mixture of experts), norms around or behind the
 * sublayers and an optional causal input convolution, every size and constant a parameter.  It owns the weights, the
 * per-sequence state (key/value caches, latent caches, retention states, convolution tails) in `max_seqs` slots, and a step function that advances any mix of sequences - whole prompts, portions of
 * prompts and single tokens - in one ragged batch.  Pure decoding replays one CUDA graph per token.
 * The reference project drives its models the same way from above (config, load by name, prompt then greedy loop:
 * mllm/Models/AutoLLM.hpp:39-105) but holds one sequence only.
 *
 * Status codes are those of mllmb200.h.  All calls are made from one thread at a time per handle.
 */
#ifndef MLLMB200_LM_H_
#define MLLMB200_LM_H_

#include "mllmb200.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { MLLMB200_LM_BF16 = 0, MLLMB200_LM_F32 = 1 };           /* activations, caches and matrix products */
enum { MLLMB200_LM_ATTENTION = 0, MLLMB200_LM_RETENTION = 1, MLLMB200_LM_LATENT = 2 }; /* mixers */
/* Gated feed-forwards, act(g) times a form of u:
 * CLAMPED: min(g, l) sigmoid(1.702 min(g, l)) (clamp(u, -l, l) + 1), l = ff_limit
 * GELU:    gelu(g) u, gelu in its tanh form;   SILU: g sigmoid(g) u */
enum { MLLMB200_LM_ACT_CLAMPED = 0, MLLMB200_LM_ACT_GELU = 1, MLLMB200_LM_ACT_SILU = 2 };
/* Norms around the sublayers:
 * SANDWICH: x + norm_b(sublayer(norm(x))), one gain per norm
 * POST:     norm(residual_scale x + sublayer(x)), one gain per column */
enum { MLLMB200_LM_NORM_SANDWICH = 0, MLLMB200_LM_NORM_POST = 1 };

typedef struct mllmb200_lm_config {
  int vocab, width, layers;
  int dtype;        /* MLLMB200_LM_BF16: bf16 matrix products with fp32 accumulation; MLLMB200_LM_F32: fp32 throughout */
  int conv_taps;    /* causal input convolution of every layer, h + conv(h); 0 = none */
  int max_seqs;     /* slots */
  int max_ctx;      /* tokens per slot */
  int max_rows;     /* tokens per step over all sequences */
  float eps;        /* of every RMS norm */
  float logit_scale;
  int norm_place;   /* MLLMB200_LM_NORM_* */
  float residual_scale; /* POST only */
  int page, pages;  /* 0: a contiguous cache of max_ctx positions per slot; else attention layers keep their keys and values in
                       `pages` pages of `page` tokens (a multiple of 16; BF16 only), which slots take as they grow */
} mllmb200_lm_config;

typedef struct mllmb200_lm_layer {
  int mixer;                 /* MLLMB200_LM_ATTENTION / MLLMB200_LM_RETENTION / MLLMB200_LM_LATENT */
  int heads, kv_heads;       /* retention and latent attention: kv_heads = heads */
  int dim, vdim;             /* per head: query/key and value size */
  float score_scale;         /* attention, latent attention: multiplies q.k (the distance bias is added after it) */
  int sink;                  /* attention: 1 = a key of score 0 without a value joins the softmax */
  int bias_rows, bias_max;   /* attention: rows of the learned distance-bias table and its largest distance; rows 0 = no bias */
  int rot_dims;              /* retention: rotated coordinates of every head, 0 = none */
  double rot_base;
  int ff;                    /* feed-forward width (of one expert), 0 = the layer has none */
  float ff_limit;            /* clamp of the gated feed-forward: min(g, limit), clamp(u, -limit, limit) */
  int weights_of;            /* -1, or the layer whose tensors this one uses (cache and state stay its own) */
  int kv_rank;               /* latent attention: cached numbers per position, from which every head's key and value are made */
  int kv_from;               /* latent attention: -1, or the earlier layer whose cached rows this one uses */
  int act;                   /* MLLMB200_LM_ACT_* */
  int experts, top;          /* mixture of experts: their number and how many a token uses; experts 0 = a dense feed-forward */
  int window, keep;          /* attention, with pages: position i sees j > i - window and j < keep alone; window 0 = everything */
} mllmb200_lm_layer;

/* Tensors of a layer; linear maps are bf16 [out, in] row-major. */
enum {
  MLLMB200_LM_T_Q = 0, MLLMB200_LM_T_K, MLLMB200_LM_T_V, MLLMB200_LM_T_G, MLLMB200_LM_T_O,
  MLLMB200_LM_T_GATE, MLLMB200_LM_T_UP, MLLMB200_LM_T_DOWN,
  MLLMB200_LM_T_NORM1, MLLMB200_LM_T_NORM1B, MLLMB200_LM_T_NORM2, MLLMB200_LM_T_NORM2B, /* fp32: one number each (SANDWICH);
                                                                                        NORM1 and NORM2, [width] (POST) */
  MLLMB200_LM_T_CONV,        /* fp32 [width, taps] */
  MLLMB200_LM_T_REL,         /* fp32 [bias_rows, heads] */
  MLLMB200_LM_T_DECAY,       /* fp64 [heads] */
  MLLMB200_LM_T_DKV,         /* latent attention: bf16 [kv_rank, width], fp32 [kv_rank], bf16 [heads dim, kv_rank], [heads vdim, kv_rank] */
  MLLMB200_LM_T_DKV_NORM, MLLMB200_LM_T_UK, MLLMB200_LM_T_UV,
  MLLMB200_LM_T_ROUTER,      /* bf16 [experts, width] */
  MLLMB200_LM_T_ROUTER_B,    /* fp32 [experts] */
  MLLMB200_LM_T_COUNT,
  /* tensors of the model (layer = -1) */
  MLLMB200_LM_T_EMBED = 100, MLLMB200_LM_T_HEAD, /* bf16 [vocab, width] */
  MLLMB200_LM_T_FINAL_NORM                       /* fp32: one number (SANDWICH) or [width] (POST) */
};

/* (Structures grow at their ends, and the symbol says which ones are meant: what was built before `page` and `window` were there calls the
 * symbol mllmb200_lm_create with structures that end in front of them.  A program that was built with `page` and the old symbol has to be
 * built again.) */
#define mllmb200_lm_create mllmb200_lm_create_paged
MLLMB200_API int mllmb200_lm_create(const mllmb200_lm_config* cfg, const mllmb200_lm_layer* layers, void** handle);
MLLMB200_API void mllmb200_lm_destroy(void* handle);

/* Loads one tensor (layer -1: a tensor of the model).  `data` may be host or device memory; rows x cols must be the
 * tensor's shape ([1, n] for a vector).  The engine keeps its own packed copy. */
MLLMB200_API int mllmb200_lm_set_tensor(void* handle, int layer, int which, const void* data, int rows, int cols);
/* The same for GATE, UP and DOWN of one expert of a mixture. */
MLLMB200_API int mllmb200_lm_set_expert(void* handle, int layer, int expert, int which, const void* data, int rows, int cols);

/* One step over `entries` sequences: entry e appends counts[e] >= 1 tokens to slot slots[e] (each slot at most once per
 * step).  tokens: all entries' tokens one after the other (host).  want: places among these sum(counts) rows whose
 * logits are copied to logits_out (host, fp32 [n_want, vocab], in the order of want).  sample != 0: the greedy next
 * token of every entry's last row is kept on the device as the slot's current token (see decode and read).
 * Synchronizes when logits are wanted.  MLLMB200_TOO_LARGE: more than max_rows rows, a slot beyond max_ctx, or more pages
 * than are free (nothing is changed then). */
MLLMB200_API int mllmb200_lm_step(void* handle, int entries, const int* slots, const int* counts, const int* tokens,
                                  int n_want, const int* want, float* logits_out, int sample);

/* The same with the probabilities of the wanted rows instead of their logits (mllmb200_lm_probabilities), to device memory, fp32
 * [n_want][ld]; nothing is sampled and nothing synchronizes: they are valid when the engine's stream reaches them. */
MLLMB200_API int mllmb200_lm_step_probabilities(void* handle, int entries, const int* slots, const int* counts, const int* tokens,
                                                int n_want, const int* want, float temperature, float* probabilities, long long ld);

/* Takes a slot back to its first `length` tokens (drafted tokens that did not stand).  MLLMB200_UNSUPPORTED where layers
 * have state that cannot go back (retention, an input convolution); MLLMB200_INVALID_ARG beyond the slot's tokens, or where
 * pages that the tokens would see again have been given up: never down to 64 tokens before the place where the slot's furthest step (or
 * decode) began, however often it is taken back meanwhile.  Nothing is changed then. */
MLLMB200_API int mllmb200_lm_truncate(void* handle, int slot, int length);

/* Pages that no slot holds (0 without pages). */
MLLMB200_API int mllmb200_lm_free_pages(void* handle, int* pages);

/* `steps` greedy steps for `count` slots together, each feeding the slot's current token; the last call on every slot
 * must have been a sampling step or a decode.  One CUDA graph replay per step. */
MLLMB200_API int mllmb200_lm_decode(void* handle, int count, const int* slots, int steps);

/* Gives a slot back: its next token is position 0 of a new sequence. */
MLLMB200_API int mllmb200_lm_free_slot(void* handle, int slot);

/* Synchronizes; history[first, first + count) of a slot (entry p = the token sampled after position p) and the number
 * of tokens it holds, to host memory; NULLs are skipped. */
MLLMB200_API int mllmb200_lm_read(void* handle, int slot, int first, int count, int* tokens_out, int* length_out);

/* Inspection: keep the residual stream after every layer of the following steps (on != 0), and read the rows of the
 * last step after `layer` (fp32 [rows, width], host). */
MLLMB200_API int mllmb200_lm_keep_residual(void* handle, int on);
MLLMB200_API int mllmb200_lm_read_residual(void* handle, int layer, int rows, float* out);

/* Bytes of per-sequence state in all slots, and kernels launched so far by steps (graph replays counted). */
MLLMB200_API int mllmb200_lm_stats(void* handle, size_t* state_bytes, long long* launches);

MLLMB200_API int mllmb200_lm_synchronize(void* handle);
MLLMB200_API void* mllmb200_lm_stream(void* handle);
MLLMB200_API const char* mllmb200_lm_last_error(void* handle);
MLLMB200_API int mllmb200_lm_check_device_status(void* handle);

/* ------------------------------------------------------------------------------------------------------------------
 * Operators on the caller's device memory, on the caller's stream and the current device: a key-value cache in pages,
 * attention of new tokens over it, and verification of drafted tokens.  They allocate nothing and never synchronize (they
 * can be captured into a CUDA graph, every call of it with a workspace of its own); results are valid when the stream
 * reaches them.  Tables, lengths and row starts are device memory and may change between replays of a graph. */

enum { MLLMB200_LM_F16 = 2 };  /* caches and queries in fp16 (beside MLLMB200_LM_BF16) */

/* A layer's cache: position j of sequence s lies in page table[s * ld_table + j / page], row j % page.  Pages may lie in
 * any order; strides are in elements (multiples of 8, whatever they are for a dimension of one; rows are contiguous), pointers
 * 16-byte aligned.
 * Sequence s brings the rows [q_start[s], q_start[s + 1]) of a call (q_start NULL: rows / seqs each) and is
 * lengths[s] tokens long with them: its row t stands at position lengths[s] - n + t.  Rows at negative positions see nothing
 * (attention: zeros) and are not stored; rows from q_start[seqs] on are neither read nor written.
 * A page number outside [0, pages): what the page would hold is taken as zeros and is not stored.  A length beyond
 * max_pages pages counts as max_pages pages in attention; rows whose position lies beyond them are not stored.  These make
 * mllmb200_lm_operator_status report MLLMB200_BAD_PAGE.  Page numbers of
 * positions that no row of the call sees are not read. */
typedef struct mllmb200_lm_pages {
  void *k, *v;                       /* dim numbers per key, vdim per value */
  long long k_page, k_head, k_row, v_page, v_head, v_row;
  const int *table, *lengths, *q_start;
  int dtype;                         /* MLLMB200_LM_BF16 or MLLMB200_LM_F16 */
  int pages, page;                   /* their number, and tokens in each: a multiple of 16 */
  int kv_heads, dim, vdim;           /* sizes: multiples of 16 up to 256 */
  int ld_table, max_pages;           /* row stride of the table, and the pages that a row names at most */
  int seqs, rows;
} mllmb200_lm_pages;

/* Attention of the rows' queries (same dtype) over the pages.  A row at position i sees key j if j <= i and (window == 0
 * or j > i - window or j < keep); scores are scale q.k + bias[h][min(i - j, bias_max)]; with `sink` the softmax of head h
 * has one more score, sink[h], without a value.  A row that sees no key gives zeros.  Scores, weights' sums and outputs are
 * summed in fp32. */
typedef struct mllmb200_lm_look {
  const void* q;                     /* [rows][heads][dim] */
  void* out;                         /* [rows][heads][vdim], not where q lies */
  long long q_row, q_head, out_row, out_head;
  const float* sink;                 /* [heads] or NULL */
  const float* bias;                 /* [heads][bias_max + 1] or NULL */
  int heads;                         /* a multiple of kv_heads, at most 64 per key head */
  int bias_max, window, keep;
  float scale;
  int exact;                         /* attn_prompt; 0 or 1, see there */
} mllmb200_lm_look;

/* New keys [rows][kv_heads][dim] and values [rows][kv_heads][vdim] into the pages (strides as above). */
MLLMB200_API int mllmb200_lm_pages_append(const mllmb200_lm_pages* pages, const void* k, long long k_row, long long k_head,
                                          const void* v, long long v_row, long long v_head, void* stream);

/* A few tokens of every sequence (q_start NULL, rows / seqs <= 16): the lengths are split over the GPU and joined. */
MLLMB200_API int mllmb200_lm_attn_decode_workspace(const mllmb200_lm_pages* pages, const mllmb200_lm_look* look, size_t* bytes);
MLLMB200_API int mllmb200_lm_attn_decode(const mllmb200_lm_pages* pages, const mllmb200_lm_look* look, void* workspace, void* stream);

/* Any number of tokens of every sequence.  Heads of 64 or 128 on the tensor cores: softmax weights are rounded to the cache's type before they
 * meet the values (half a step of every weight, an error of the size of the outputs' own rounding), or, look->exact, carried by two numbers of it
 * (2^-16 and better; a third more time on long prompts).  attn_decode and all other head sizes always carry two. */
MLLMB200_API int mllmb200_lm_attn_prompt_workspace(const mllmb200_lm_pages* pages, const mllmb200_lm_look* look, size_t* bytes);
MLLMB200_API int mllmb200_lm_attn_prompt(const mllmb200_lm_pages* pages, const mllmb200_lm_look* look, void* workspace, void* stream);

/* Rows of logits to probabilities: exp((z - max z) / temperature) over their sum; temperature 0: 1 at the first largest.
 * -inf gives 0; a row of nothing but -inf, zeros; a row with NaN or +inf, NaN (temperature 0: NaN is passed over).
 * dtype: MLLMB200_LM_F32, _BF16 or _F16; out fp32.  vocab: at most 2^30. */
MLLMB200_API int mllmb200_lm_probabilities(const void* logits, int dtype, long long ld, int rows, int vocab, float temperature,
                                           float* out, long long ld_out, void* stream);

/* Drafted tokens against the target's probabilities.  target: fp32 [seqs][drafts + 1][vocab], draft: fp32
 * [seqs][drafts][vocab], tokens: [seqs][drafts], accept: uniform numbers in [0, 1) per draft, pick: one per sequence.  Token x
 * at place i is accepted while accept q(x) < p(x) (products and sums in 64 bits); at the first refused place the next token
 * comes from max(p - q, 0) (from p where that has no mass), behind the last draft from p: the lowest index whose running sum
 * exceeds pick times the whole.  A token outside [0, vocab) ends a sequence's drafts: the next token comes from p there.
 * Negative numbers and NaN count as 0.  accepted[s]: accepted drafts; out [seqs][drafts + 1]: these, the next token (-1 where
 * p has no mass), and -1 behind it.  drafts may be 0: a plain draw from p.  vocab: at most 2^20. */
MLLMB200_API int mllmb200_lm_verify(const float* target, long long t_seq, long long t_row, const float* draft, long long d_seq,
                                    long long d_row, const int* tokens, long long ld_tokens, const float* accept,
                                    long long ld_accept, const float* pick, int seqs, int drafts, int vocab, int* accepted,
                                    int* out, long long ld_out, void* stream);

/* Waits for the stream; reads and clears what these operators found wrong on the current device, on any stream (calls that are
 * checked one by one are checked before the next is made).  One kind a call: another that was found is told by the next.
 * The engines' status (mllmb200_lm_check_device_status) is apart from this. */
MLLMB200_API int mllmb200_lm_operator_status(void* stream);

/* Host only: the distance buckets of a bias table, out[n] for n in [0, count). */
MLLMB200_API int mllmb200_lm_distance_buckets(int bias_rows, int bias_max, int count, int* out);

#ifdef __cplusplus
}
#endif
#endif /* MLLMB200_LM_H_ */
