/*
 * dsa_vocab.h — C ABI of the operators on a vocabulary's logits in libdsa.so:
 *
 *   token log probabilities   z = logits / T, lse = log sum_j exp(z_j):
 *       logprob = z_id - lse, entropy = -sum_j p_j log p_j, lse, and the k
 *       largest z with their z - lse; the gradient of all of them.
 *       The generator's loss over masked positions, scoring, answers.
 *   distillation loss         T^2 sum_t q_t (log q_t - (z_{id_t} - lse)) for a
 *       teacher's entries (id_t, logit_t), q their softmax at T; its gradient.
 *
 * Conventions are those of dsa.h: the caller owns every buffer, work goes on
 * the caller's stream, a nonzero return carries a message in dsa_last_error().
 * Rows (2^36 at most) hold V contiguous values; the logits' and the gradient's
 * row strides are given, every other tensor is contiguous, and what a call writes
 * overlaps nothing else that it takes.  Logits are DSA_F32 or DSA_BF16;
 * arithmetic, sums and results are float32.  Equal calls give equal bits (no
 * float atomics).  The order of a row's sums goes by where it begins between two
 * 128-byte borders, by N, V and dtype and by whether top_k is 0: other rows beside
 * it, or the largest asked for, may change the last bits of its results.
 *
 * A logit of -inf has probability 0 and adds nothing to sums, entropy or
 * gradients.  A row with a NaN or +inf among its logits, or without a finite
 * one, has NaN results (lse -inf in a row of -inf alone).  Among the largest
 * NaN counts as -inf and -0 as +0; equal values go by their lower index.
 */
#ifndef DSA_VOCAB_H_
#define DSA_VOCAB_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum {
  DSA_VOCAB_MAX_ENTRIES = 128,     /* largest values, or a teacher's entries, of a row */
  DSA_VOCAB_MAX_TOP_V = 1 << 19    /* columns of a call that asks for the largest */
};

typedef struct dsa_logprobs_args {
  /* forward inputs */
  const void* logits;         /* [N, V], row stride logits_stride (0 and more; rows may overlap) */
  int64_t logits_stride;
  const void* ids;            /* [N] given tokens, int32 or int64 (ids_bytes), or NULL */
  int64_t ignore_index;       /* a row with this id: results 0, top ids -1, gradient 0 */
  /* results; each may be NULL in the forward but stats, where a backward follows */
  float* logprobs;            /* [N]; NaN where the id is outside [0, V) */
  float* entropy;             /* [N] */
  float* lse;                 /* [N] */
  float* top_logprobs;        /* [N, top_k], with top_ids */
  int64_t* top_ids;           /* [N, top_k]; read by the backward with dtop */
  float* stats;               /* [N, 4], 16-byte aligned; written by the forward, read by the backward */
  /* the backward's: gradients of the results, each NULL or contiguous; a stride
     of 0 reads one value for all rows */
  const float* dlogprobs;
  const float* dentropy;
  const float* dlse;
  const float* dtop;          /* [N, top_k] */
  int64_t dlogprobs_stride, dentropy_stride, dlse_stride; /* 0 or 1 */
  void* dlogits;              /* [N, V] in the logits' type, row stride dlogits_stride */
  int64_t dlogits_stride;
  void* workspace;            /* the forward's, 16-byte aligned */
  size_t workspace_bytes;
  int64_t N;
  int64_t V;
  int32_t top_k;              /* 0 .. min(V, DSA_VOCAB_MAX_ENTRIES) */
  int32_t ids_bytes;          /* 4 or 8 */
  int32_t dtype;              /* of logits and dlogits */
  float inv_temperature;      /* 1 / T, in [2^-100, 2^100] */
} dsa_logprobs_args;

typedef struct dsa_distill_args {
  const void* logits;         /* [N, V] */
  int64_t logits_stride;
  const void* teacher_ids;    /* [N, K], int32 or int64 (ids_bytes); negative: no entry */
  const void* teacher;        /* [N, K] logits, teacher_dtype */
  const float* teacher_lse;   /* [N] or NULL: q = exp(teacher / T - teacher_lse) in place of the softmax */
  float* loss;                /* [N]; 0 without an entry, NaN where an id is V or more */
  float* stats;               /* [N, 4], 16-byte aligned, as above */
  const float* dloss;         /* [N] */
  int64_t dloss_stride;       /* 0 or 1 */
  void* dlogits;
  int64_t dlogits_stride;
  void* workspace;            /* the forward's */
  size_t workspace_bytes;
  int64_t N;
  int64_t V;
  int32_t K;                  /* 1 .. DSA_VOCAB_MAX_ENTRIES */
  int32_t ids_bytes;
  int32_t dtype;
  int32_t teacher_dtype;
  float temperature;          /* in [2^-100, 2^100] */
} dsa_distill_args;

/* Workspace bytes of a forward on N rows of V values of `dtype`, with the top_k
 * largest (0 for none and for the distillation loss).  May be 0; the calls refuse
 * a smaller workspace. */
size_t dsa_vocab_workspace_bytes(int64_t N, int64_t V, int32_t dtype, int32_t top_k);

/* logprobs, entropy, lse, the largest and stats from logits and ids. */
int dsa_logprobs_fwd(const dsa_logprobs_args* args, void* stream);
/* dlogits from the results' gradients and the forward's logits, ids, top_ids
 * and stats.  With an id outside [0, V) and a gradient of its log probability
 * that is not 0 the row is NaN. */
int dsa_logprobs_bwd(const dsa_logprobs_args* args, void* stream);

/* loss and stats from logits and the teacher's entries. */
int dsa_distill_fwd(const dsa_distill_args* args, void* stream);
/* dlogits from dloss, the forward's inputs and stats; entries with one id add up. */
int dsa_distill_bwd(const dsa_distill_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DSA_VOCAB_H_ */
