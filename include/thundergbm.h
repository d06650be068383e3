/*
 * C ABI of libthundergbm.so (B200 / sm_100a build of the histogram tree-building path).
 *
 * Part 1 is the reference's own `extern "C"` surface: the functions its Python wrapper binds
 * through ctypes (python/thundergbm/thundergbm.py) and its R wrapper through .C (R/gbm.R).
 * Names, argument order and argument meaning are the reference's.  Where the reference declares
 * `Tree *&model` the ABI is a pointer to the handle, written `Tree **` here.
 *
 * Part 2 is an explicit-state interface to the same path (create / boost / read back) used by the
 * benchmark, by multi-GPU launches (one process per GPU) and by the parity tests.
 *
 * Every entry point works on plain pointers and sizes; all device memory is owned by the library.
 * Functions of part 1 return void like the reference; on failure they log the message, leave
 * `*model` NULL (the Python wrapper tests for that) and keep it for tgbm_last_error().
 */
#ifndef THUNDERGBM_B200_H
#define THUNDERGBM_B200_H

#ifdef __cplusplus
extern "C" {
#endif

typedef struct Tree Tree; /* opaque: one tree = 2^(depth+1)-1 node records of 48 bytes */

/* ---------------------------------------------------------------- part 1: reference surface */

/* src/thundergbm/scikit_tgbm.cpp:13-23 -- 0 silent, 1 info, 2 debug */
void set_logger(int verbose);

/* src/thundergbm/scikit_tgbm.cpp:26-80.  CSR is borrowed (copied inside); `col_ptr` is the column
 * index array.  Out: *model = new Tree[n_trees * *tree_per_iter] (free with model_free), *num_class,
 * *tree_per_iter, group_label[0..n_labels). */
void sparse_train_scikit(int row_size, float *val, int *row_ptr, int *col_ptr, float *label, int depth, int n_trees,
                         int n_device, float min_child_weight, float lambda, float gamma, int max_num_bin, int verbose,
                         float column_sampling_rate, int bagging, int n_parallel_trees, float learning_rate,
                         char *obj_type, int *num_class, char *tree_method, Tree **model, int *tree_per_iter,
                         float *group_label, int *group, int num_group);

/* src/thundergbm/scikit_tgbm.cpp:83-121.  y_pred: row_size floats (row_size*num_class, class-major, for
 * multi:softprob), after the objective's predict_transform.  base_score is not applied on this path. */
void sparse_predict_scikit(int row_size, float *val, int *row_ptr, int *col_ptr, float *y_pred, Tree **model,
                           int n_trees, int trees_per_iter, char *objective, int num_class, float learning_rate,
                           float *group_label, int *group, int num_group, int verbose);

/* src/thundergbm/scikit_tgbm.cpp:123-146 -- writes the reference's binary model file (src/thundergbm/parser.cpp:146-171) */
void save(char *model_path, char *objective, float learning_rate, int num_class, int n_trees, int trees_per_iter,
          Tree **model, float *group_label);
/* src/thundergbm/scikit_tgbm.cpp:148-171 */
void load_model(char *model_path, float *learning_rate, int *num_class, int *n_trees, int *trees_per_iter, Tree **model);
/* src/thundergbm/scikit_tgbm.cpp:173-182 */
void load_config(char *model_path, float *group_label);
/* src/thundergbm/scikit_tgbm.cpp:184-197 */
void get_n_nodes(Tree **model, int *n_nodes, int n_trees, int tree_per_iter);
/* src/thundergbm/scikit_tgbm.cpp:199-248 */
void get_a_tree(Tree **model, int tree_id, int n_nodes, int *children_left, int *children_right, int *children_default,
                int *features, float *thresholds, float *values, float *node_sample_weights);
/* src/thundergbm/scikit_tgbm.cpp:250-254 */
void model_free(Tree **model);

/* src/thundergbm/gbm_R_interface.cpp:10-61 and :63-87 (.C calling convention: every argument a pointer) */
void train_R(int *depth, int *n_trees, int *n_gpus, int *verbose, int *profiling, char **data, int *max_num_bin,
             double *column_sampling_rate, int *bagging, int *n_parallel_trees, double *learning_rate, char **objective,
             int *num_class, int *min_child_weight, double *lambda_tgbm, double *gamma, char **tree_method,
             char **model_out);
void predict_R(char **data, char **model_in, int *verbose);

/* ---------------------------------------------------------------- part 2: explicit-state interface */

typedef struct TgbmBooster TgbmBooster;
typedef struct TgbmComm TgbmComm;

typedef struct {
    int depth, n_trees, max_num_bin, num_class;
    float min_child_weight, lambda, gamma, learning_rate;
    const char *objective;
    int quant_bits;     /* value bits of the fixed-point gradient grid (default 18) */
    int keep_nid;       /* keep the final node id of every row for every tree (tests) */
    int verbose;
    int profile;        /* time the histogram and partition kernels with CUDA events */
    unsigned rank_seed; /* LambdaRank partner sampling */
    int hist_mode;      /* histogram arithmetic: 0 fp32 -- sums of the float (g,h): in the first round added value by value
                           into one float accumulator per bin, what the reference does in every round
                           (hist_tree_builder_single.cu:203-216, :485-505); in later rounds integer sums of the gradients, each
                           rounded by at most 2^-30 of the round's largest, as long as that is no worse than float sums;
                           rounds whose gradients differ too much in size for it sum floats as in the first;
                           1 exact -- integer sums on a fixed-point grid in every round, bit-identical from run to run and
                           for any number of GPUs */
    int bagging;        /* RowSampler::do_bagging (src/thundergbm/row_sampler.cu:9-35): bootstrap multiplicities on (g,h) */
    float column_sampling_rate; /* Shard::column_sampling (src/thundergbm/builder/shard.cu:8-23); 1 = off */
    unsigned sample_seed;       /* seed of both samplers (the reference draws from std::rand()) */
    int column_shards;  /* 0: cut points, candidate order and child sums of HistTreeBuilder_single, the reference's builder
                           for n_device = 1; D >= 1: those of the column-sharded HistTreeBuilder it runs for n_device = D > 1
                           (src/thundergbm/builder/hist_tree_builder.cu, hist_cut.cu:104-187), whose cut points depend on D */
    int exact_builder;  /* 1: tree_method = exact, the reference's ExactTreeBuilder (src/thundergbm/builder/exact_tree_builder.cu):
                           every distinct stored value of a node is a split candidate; one GPU */
} TgbmParam;

typedef struct {
    int n_rows, n_features, fpad, n_bins, trees_per_round, n_nodes, num_class, rounds_done, n_labels;
    float base_score;
    int csr_layout; /* 1: wide sparse data kept as CSR of global bin ids, 0: dense byte matrices */
} TgbmInfo;

typedef struct {
    double hist_ms, hist_bytes, hist_root_ms, hist_root_bytes, partition_ms, partition_bytes;
    long long hist_launches, hist_root_launches, partition_launches, kernel_launches;
    long long hist_rows; /* rows the timed histogram launches processed */
} TgbmProfile;

/* message of the last failure on this thread ("" if none) */
const char *tgbm_last_error(void);
void tgbm_default_param(TgbmParam *p);

/* one process per GPU: rank 0 makes the id, every rank calls create with it (NCCL underneath) */
int tgbm_comm_unique_id(unsigned char id[128]);
TgbmComm *tgbm_comm_create(const unsigned char id[128], int rank, int world);
void tgbm_comm_destroy(TgbmComm *c);

/* Booster::init (include/thundergbm/booster.h:36-74): CSR rows of THIS rank -> cut points, bin matrix, base score.
 * `comm` may be NULL.  Returns NULL on failure. */
TgbmBooster *tgbm_booster_create(int n_rows, const float *val, const int *row_ptr, const int *col, const float *label,
                                 const int *group, int num_group, const TgbmParam *param, TgbmComm *comm);
/* Booster::boost x n_rounds; queues the work on the booster's stream and returns */
int tgbm_booster_boost(TgbmBooster *b, int n_rounds);
/* Objectives multi:softmax and multi:softprob, before the first round: trees are grown on the pairs of tgbm_scores_distill (below) instead of
 * the hard labels' alone -- per row of this rank `top` classes and scores of a teacher, its log-sum-exp at `temperature` (or NULL), the
 * labels' part weighing 1 - alpha.  Host arrays n_rows x top, n_rows x top, n_rows; copied.  Classes are positions among the labels
 * (tgbm_booster_get_labels).  With a communicator every rank calls it, with the same temperature and alpha and all with lse or none; where
 * one rank's call is refused, all are, and what was set before stays.  Metrics stay those of the labels; model files do not change. */
int tgbm_booster_set_teacher(TgbmBooster *b, int top, const int *ids, const float *logits, const float *lse, float temperature, float alpha);
/* The same from classes that were drawn for the rows and the gains that followed: trees are grown on the pairs of tgbm_scores_feedback (below,
 * without a reference) instead of the labels'.  Host arrays n_rows x draws (old: or NULL), weights n_rows (or NULL); copied.  Not beside a teacher.
 * Ranks call it together, as above, with the same temperature, clip and entropy and all with old and weights or none. */
int tgbm_booster_set_feedback(TgbmBooster *b, int draws, const int *classes, const float *gains, const float *old, const float *weights, float temperature,
                              float clip_low, float clip_high, float entropy);
/* those losses on the current scores: their mean over this rank's rows (wait as tgbm_booster_sync does; with a communicator every rank calls them) */
int tgbm_booster_teacher_loss(TgbmBooster *b, double *out);
int tgbm_booster_feedback_loss(TgbmBooster *b, double *out);
int tgbm_booster_sync(TgbmBooster *b);
/* boost + sync, bracketed by CUDA events on the booster's stream: device time of the n_rounds in ms */
int tgbm_booster_boost_timed(TgbmBooster *b, int n_rounds, float *elapsed_ms);
/* switch the per-kernel CUDA-event timing of the histogram and partition kernels on or off */
int tgbm_booster_set_profile(TgbmBooster *b, int on);
int tgbm_booster_info(TgbmBooster *b, TgbmInfo *out);
int tgbm_booster_profile(TgbmBooster *b, TgbmProfile *out);
/* rounds_done * trees_per_round * n_nodes records of 48 bytes */
int tgbm_booster_get_trees(TgbmBooster *b, void *nodes_out);
int tgbm_booster_get_metrics(TgbmBooster *b, float *out);            /* rounds_done */
int tgbm_booster_get_ypred(TgbmBooster *b, float *out);              /* trees_per_round * n_rows */
int tgbm_booster_get_cuts(TgbmBooster *b, float *cut_val, int *cut_ptr); /* n_bins, n_features+1 */
int tgbm_booster_get_bins(TgbmBooster *b, unsigned char *out);       /* dense layout: n_rows * fpad, 255 = missing */
int tgbm_booster_get_bins_csr(TgbmBooster *b, int *out);             /* CSR layout: global bin id per stored value */
int tgbm_booster_get_nid(TgbmBooster *b, int *out);                  /* rounds_done*trees_per_round*n_rows (keep_nid) */
int tgbm_booster_get_root_hist(TgbmBooster *b, long long *out);      /* exact mode: n_bins*2 of the last tree */
int tgbm_booster_get_root_hist_f32(TgbmBooster *b, float *out);      /* fp32 mode: n_bins*2 of the last tree */
int tgbm_booster_get_quant_scale(TgbmBooster *b, double *out);       /* rounds_done*2 */
int tgbm_booster_get_labels(TgbmBooster *b, float *out);             /* n_labels */
/* hands the trained trees over as the opaque model of part 1 */
int tgbm_booster_to_model(TgbmBooster *b, Tree **model);
void tgbm_booster_free(TgbmBooster *b);
/* The library's device buffers come from one memory pool per GPU that keeps what a call releases (up to
 * TGBM_POOL_KEEP_MB megabytes, default 16384; TGBM_NO_POOL=1: plain cudaMalloc / cudaFree), so that the next call finds
 * its memory mapped.  This gives every unused block back to the driver now. */
void tgbm_release_device_memory(void);

/* Predictor::predict_raw (src/thundergbm/predictor.cu:32-189) on node records as returned by
 * tgbm_booster_get_trees: out[t * n_rows + i] */
int tgbm_predict_raw(int n_rows, const float *val, const int *row_ptr, const int *col, const void *nodes, int n_rounds,
                     int trees_per_round, int n_nodes, float learning_rate, float base_score, float *out);
/* the same, also returning the device time of the traversal kernel alone (measurement) */
int tgbm_predict_raw_timed(int n_rows, const float *val, const int *row_ptr, const int *col, const void *nodes, int n_rounds,
                     int trees_per_round, int n_nodes, float learning_rate, float base_score, float *out, float *kernel_ms);

/* sparse_train_scikit / sparse_predict_scikit on a row-major matrix of floats (is_f64 = 0) or doubles (is_f64 = 1) in host
 * memory, n_rows x n_cols with n_rows * n_cols < 2^31.  A zero is not stored, as in the CSR scipy.sparse.csr_matrix makes of
 * the matrix: results are those of the two functions above on that CSR, which is made on the GPU. */
void dense_train_scikit(int row_size, int n_cols, void *x, int is_f64, float *label, int depth, int n_trees,
                        int n_device, float min_child_weight, float lambda, float gamma, int max_num_bin, int verbose,
                        float column_sampling_rate, int bagging, int n_parallel_trees, float learning_rate,
                        char *obj_type, int *num_class, char *tree_method, Tree **model, int *tree_per_iter,
                        float *group_label, int *group, int num_group);
void dense_predict_scikit(int row_size, int n_cols, void *x, int is_f64, float *y_pred, Tree **model,
                          int n_trees, int trees_per_iter, char *objective, int num_class, float learning_rate,
                          float *group_label, int verbose);
/* number of distinct values (every NaN counts, +0 and -0 are one): the labels a group_label buffer must have room for;
 * -1 when there is no memory to count them in (tgbm_last_error()) */
int tgbm_count_distinct(const float *v, long long n);
/* The same on a thread of its own.  `v` is read until tgbm_count_distinct_wait() returns, which gives the number and frees the
 * handle; null / -1: as above. */
void *tgbm_count_distinct_start(const float *v, long long n);
int tgbm_count_distinct_wait(void *count);

/* Metric::get_score of the objective's default metric (the .cu files under src/thundergbm/metric, rank_metric.cpp) on raw scores
 * raw[t * n_rows + i]: RMSE, binary error, multi-class accuracy, MAP or NDCG.  `label` holds class indices for the
 * classification objectives.  Host pointers; device buffers and reduction scratch are allocated inside. */
int tgbm_metric_score(const char *objective, int n_rows, int trees_per_round, const float *label, const float *raw,
                      const int *group, int num_group, float *out);

/* The same metric for callers that must not allocate device memory: a host whose own pool already owns the whole
 * GPU, or a hook inside another program's step loop that cannot afford the device-wide synchronisation of
 * cudaMalloc / cudaFree.  No counterpart in the reference (every reference entry point allocates).
 * d_label, d_raw (raw[t * n_rows + i]) and d_out (one float) are DEVICE pointers owned by the caller; the kernels
 * are queued on `cuda_stream` (a cudaStream_t, NULL = default stream) and the call returns without waiting.
 * The reduction scratch is a fixed 8.2 KB array inside the library image on every GPU that loads the library.
 * n_rows <= TGBM_NOALLOC_MAX_ROWS, trees_per_round <= TGBM_NOALLOC_MAX_CLASSES, no ranking objectives; anything else
 * returns 1 with the reason in tgbm_last_error().  The first call on each device resolves the scratch address and
 * should be made outside stream capture.  All calls on a device share the scratch: calls whose kernels can overlap
 * on the GPU (unordered streams) race; calls on one stream are safe. */
#define TGBM_NOALLOC_MAX_ROWS (1 << 30)
#define TGBM_NOALLOC_MAX_CLASSES 1024
int tgbm_metric_score_noalloc(const char *objective, int n_rows, int trees_per_round, const float *d_label,
                              const float *d_raw, float *d_out, void *cuda_stream);

/* ---- operators on the scores of many classes (no counterpart in the reference) ----
 * All pointers whose names begin with d_ are DEVICE pointers of the caller, on the current device; the kernels are queued on
 * `cuda_stream` (a cudaStream_t, NULL = default stream) and the calls return without waiting.  Nothing is allocated and nothing is
 * kept from one call for the next: calls on different streams do not disturb each other, and a call may be captured into a graph.
 * Arguments are checked before anything is queued: 1 and a message in tgbm_last_error().  No result may share memory with what is read
 * or with another result, except where it is said to work (adjust and norm refuse it for what they read, distill, feedback and norm_backward for scores
 * and gradients; the rest is the caller's to see to).
 * Scores are a matrix of n_rows x n_classes in `type`, class k of row n at d_scores[n * row_stride + k * class_stride] (strides in
 * elements, none negative).  Row stride 1: by class, as tgbm_booster_get_ypred and tgbm_predict_raw lay them out; class stride 1:
 * by row, as networks do.  Where neither is 1 the operators work as well, more slowly, and so do top and distill by class above some 5000
 * classes (scores of 2000 x 10000 13 and 4 times as long as of 4000 x 5000), and sample, feedback, norm and norm_backward by class above 1024
 * (4000 x 5000: up to 9 times as long as by row).  How far a score lies below the largest of its row is a float (in sample a double): infinite beyond
 * 3.4e38. */
#define TGBM_F32 0
#define TGBM_F16 1
#define TGBM_BF16 2
#define TGBM_SCORES_MAX_CLASSES (1 << 20)
#define TGBM_SCORES_MAX_TOP 128

/* Scores as a user's rules change them before classes are chosen.  For class k of row n, with c the number of times it stands in
 * the row's history:
 *   z = c > 0 ? (s > 0 ? s / repetition : s * repetition) : s;   z -= c * frequency + (c > 0 ? presence : 0);
 *   z += d_bias[k];   out = allowed ? z : -infinity
 * computed in floats and rounded once (repetition > 0, and a float holds 1 / repetition).  d_out: the same type, strides of its own;
 * d_out = d_scores with the same strides works in place; otherwise the two must not share memory (and where their lines interleave
 * with gaps between the cells of a line, the call is refused although they do not).
 * d_bias: n_classes floats, or NULL.
 * d_allowed: n_masks rows of at least (n_classes + 31) / 32 words, `mask_stride` words apart, class k in bit k & 31 of word k >> 5;
 * NULL: every class is allowed.  d_allowed_row[n]: the row's mask (outside [0, n_masks): all its classes are allowed); NULL: row n
 * has mask n.
 * d_history[d_history_ptr[n] .. d_history_ptr[n + 1]): classes given before, repeated as often as they were, in any order; numbers
 * outside [0, n_classes) are passed over.  d_history_ptr has n_rows + 1 entries, d_history n_history; NULL: no histories. */
int tgbm_scores_adjust(int n_rows, int n_classes, int type, const void *d_scores, long long row_stride, long long class_stride, void *d_out,
                       long long out_row_stride, long long out_class_stride, const float *d_bias, const unsigned *d_allowed, int n_masks,
                       long long mask_stride, const int *d_allowed_row, const long long *d_history_ptr, const int *d_history,
                       long long n_history, float repetition, float frequency, float presence, void *cuda_stream);

/* The `top` largest scores of every row, 1 <= top <= TGBM_SCORES_MAX_TOP: d_values and d_ids are n_rows x top, largest first, of
 * equal scores the lower class first.  -infinity (masked) and NaN are never chosen; where a row has fewer than `top` other scores
 * the last entries are -infinity and class -1.  d_lse (n_rows floats, or NULL): log of the sum over ALL classes of
 * exp(score / temperature), so that value / temperature - lse is the log of a class's share; NaN where a score is NaN or +infinity. */
int tgbm_scores_top(int n_rows, int n_classes, int type, const void *d_scores, long long row_stride, long long class_stride, int top,
                    float temperature, float *d_values, int *d_ids, float *d_lse, void *cuda_stream);

/* Distance of a student's scores s from what is kept of a teacher: per row `top` classes d_ids and their scores d_logits t (type
 * logits_type; rows ids_stride and logits_stride elements apart).  With T the temperature, p = softmax(s / T):
 *   q_j = exp(t_j / T - L);  L = d_lse[n], the teacher's log-sum-exp over all classes AT THIS T (what tgbm_scores_top gives), and
 *   the mass that is not listed, r = max(0, 1 - sum q), lies on the unlisted classes together; d_lse NULL: L = log sum exp(t_j / T)
 *   over the listed ones, r = 0.
 *   loss = w (alpha T^2 (sum q_j log(q_j / p_j) + r log(r / p_r)) - (1 - alpha) log softmax(s)_y)
 * with p_r the student's share of the unlisted classes, w = d_weights[n] (NULL: 1) and y = d_labels[n] (outside [0, n_classes), or
 * NULL: no such term).  A class number outside [0, n_classes) is passed over, one that stands twice in a row holds the sum; a row
 * that lists nothing, or only -infinity, has no teacher: its first term is 0.  What weighs 0 (a term by alpha, a row by w) counts for
 * nothing, also where it is infinite, and so does a class to which the teacher gives less than a float holds (e^-103 of its mass).
 * d_loss: n_rows floats (NULL: not wanted, where there is a gradient).
 * gives: TGBM_GIVES_LOSS; TGBM_GIVES_GRADIENT: d_grad holds d loss / d s in the type of the scores; TGBM_GIVES_PAIRS: pairs of floats
 * (gradient, hessian) as a booster takes them, hessian = max(2 w (alpha p (1 - p) + (1 - alpha) p1 (1 - p1)), 1e-16), p1 = softmax(s), each
 * term where the row has it -- with alpha = 0 the pairs of the objective multi:softmax; the unlisted classes' share of the first term's
 * second derivative that could make it negative is left out.  Strides of d_grad in elements (pairs). */
#define TGBM_GIVES_LOSS 0
#define TGBM_GIVES_GRADIENT 1
#define TGBM_GIVES_PAIRS 2
int tgbm_scores_distill(int n_rows, int n_classes, int type, const void *d_scores, long long row_stride, long long class_stride, int top,
                        const int *d_ids, long long ids_stride, int logits_type, const void *d_logits, long long logits_stride,
                        const float *d_lse, const int *d_labels, const float *d_weights, float temperature, float alpha, float *d_loss,
                        int gives, void *d_grad, long long grad_row_stride, long long grad_class_stride, void *cuda_stream);

/* Classes drawn from the scores s of every row, one for each of `draws` given random numbers u (1 to TGBM_SCORES_MAX_DRAWS per row; d_uniform is
 * n_rows x draws of uniform_type TGBM_F32 or TGBM_F64, in [0, 1): numbers outside are taken as the nearest double inside, NaN as 0).
 *   w_k = exp((s_k - max s) / temperature) for every class whose score is above -infinity
 *   A: classes with w_k >= min_p that are among the top_k largest scores (of equal ones the lower class first; 0: all)
 *   B: the shortest beginning of A, largest first, whose mass is at least top_p of A's (never empty; top_p 1: all of A)
 *   a draw is the first class k of B in class order up to which B's mass goes beyond u times B's whole mass
 * d_classes: n_rows x draws.  d_logs (or NULL): log of the drawn class's share of B's mass; d_all_logs (or NULL): of all classes' mass.
 * temperature 0: the largest score (the lower class of equal ones), both logs 0.  A row without a score above -infinity gives class -1 and
 * logs of -infinity, one that holds NaN or +infinity class -1 and NaN.
 * Each of the four limits holds for all rows, or (where d_temperature, d_top_k, d_top_p, d_min_p is not NULL) is read per row: a temperature
 * that is negative or no finite number gives class -1 and NaN, top_k below 1, top_p above 1 or NaN and min_p below 0 or NaN limit
 * nothing.  Masses are sums of doubles, of exponentials good to 2^-38. */
#define TGBM_F64 3
#define TGBM_SCORES_MAX_DRAWS 128
int tgbm_scores_sample(int n_rows, int n_classes, int type, const void *d_scores, long long row_stride, long long class_stride, int draws,
                       int uniform_type, const void *d_uniform, float temperature, const float *d_temperature, int top_k, const int *d_top_k,
                       float top_p, const float *d_top_p, float min_p, const float *d_min_p, int *d_classes, float *d_logs, float *d_all_logs,
                       void *cuda_stream);

/* Loss on classes that were drawn, `draws` per row, and on the gains that followed: with T the temperature, p = softmax(s / T),
 *   l = log p[class];  r = exp(l - d_old) (d_old NULL: 1, as if drawn now);  held r: r within [1 - clip_low, 1 + clip_high]
 *   loss = w (mean over the row's draws that count of (-min(r gain, held r gain) + kl (exp(x) - x - 1)) - entropy H)
 * with x = d_reference - l, H = -sum p log p and w = d_weights[n] (NULL: 1).  d_classes, d_gains, d_old, d_reference and d_logs are n_rows x draws.
 * A draw counts unless its class lies outside [0, n_classes) or its score is -infinity; a row without one has loss 0 and no gradient.  What
 * weighs 0 (a gain, kl, entropy, a row by w) counts for nothing.  clip_low 1 and clip_high infinity: r is not held.  kl above 0 needs d_reference.
 * d_loss: n_rows floats, or NULL; d_logs (or NULL): l, -infinity where the draw does not count.
 * gives: as for tgbm_scores_distill; pairs have hessian = max(2 w / T^2 (mean |d loss of a draw / d l| + entropy) p (1 - p), 1e-16). */
int tgbm_scores_feedback(int n_rows, int n_classes, int type, const void *d_scores, long long row_stride, long long class_stride, int draws,
                         const int *d_classes, const float *d_gains, const float *d_old, const float *d_reference, const float *d_weights,
                         float temperature, float clip_low, float clip_high, float kl, float entropy, float *d_loss, float *d_logs, int gives,
                         void *d_grad, long long grad_row_stride, long long grad_class_stride, void *cuda_stream);

/* Every row at mean 0 and variance 1 over its classes, then a gain and a bias per class:
 *   out_k = (s_k - mean) rstd gain_k + bias_k,  rstd = 1 / sqrt(variance + eps)
 * over the classes whose score is not -infinity; those stay -infinity.  A row without another class has mean 0 and rstd 0.  Sums are floats: where
 * the squared deviations add up to more than one holds (scores some 1e19 apart) rstd is 0, where the scores do mean is not finite.  d_out: the type
 * of the scores, strides of its own; d_out = d_scores with the same strides works in place, otherwise the two must not share memory.
 * d_gain, d_bias: n_classes floats, NULL: 1, 0.  d_mean, d_rstd: n_rows floats, or NULL.  eps > 0. */
int tgbm_scores_norm(int n_rows, int n_classes, int type, const void *d_scores, long long row_stride, long long class_stride, void *d_out,
                     long long out_row_stride, long long out_class_stride, const float *d_gain, const float *d_bias, float eps, float *d_mean,
                     float *d_rstd, void *cuda_stream);

/* The way back: with x_k = (s_k - mean) rstd and g the gradient of out (`d_grad`, the type of the scores), a_k = g_k gain_k,
 *   d_out_k = rstd (a_k - mean(a) - x_k mean(a x));  d_grad_gain_k = sum over rows of g_k x_k;  d_grad_bias_k = sum over rows of g_k
 * means over the classes that the row may have; where a score is -infinity g is not looked at and d_out is 0.  d_mean, d_rstd: from
 * tgbm_scores_norm.  d_grad_gain and d_grad_bias: n_classes floats, both or both NULL; where they are wanted, d_work is memory of at least
 * tgbm_scores_norm_work(n_rows, n_classes) bytes, aligned to 16, of which nothing is kept.  Sums are made in the same order every time.
 * d_out may not share memory with d_grad or d_scores. */
long long tgbm_scores_norm_work(int n_rows, int n_classes);
int tgbm_scores_norm_backward(int n_rows, int n_classes, int type, const void *d_grad, long long grad_row_stride, long long grad_class_stride,
                              const void *d_scores, long long row_stride, long long class_stride, const float *d_mean, const float *d_rstd,
                              const float *d_gain, void *d_out, long long out_row_stride, long long out_class_stride, float *d_grad_gain,
                              float *d_grad_bias, void *d_work, long long work_bytes, void *cuda_stream);

/* A model's raw scores (as sparse_predict_scikit and dense_predict_scikit compute them, before the objective's transformation) through
 * tgbm_scores_adjust and tgbm_scores_top, from and to HOST arrays: the `top` best classes of every row under the caller's rules.  For models of
 * several classes (trees_per_iter >= 2); classes are positions among the model's labels.  rules NULL: none.  values and ids: row_size x
 * top; lse (or NULL): row_size. */
typedef struct {
    const float *bias;            /* one per class, or NULL */
    const unsigned *allowed;      /* n_masks x (classes + 31) / 32 words, or NULL */
    int n_masks;
    const int *allowed_row;       /* mask of every row, or NULL: row n has mask n */
    const long long *history_ptr; /* row_size + 1, or NULL */
    const int *history;
    float repetition, frequency, presence; /* 1, 0, 0: no penalty */
} TgbmTopRules;
int tgbm_predict_top(int row_size, float *val, int *row_ptr, int *col_ptr, Tree **model, int n_trees, int trees_per_iter, float learning_rate,
                     const TgbmTopRules *rules, int top, float temperature, float *values, int *ids, float *lse);
int tgbm_predict_top_dense(int row_size, int n_cols, void *x, int is_f64, Tree **model, int n_trees, int trees_per_iter, float learning_rate,
                           const TgbmTopRules *rules, int top, float temperature, float *values, int *ids, float *lse);
/* The same scores through tgbm_scores_adjust and tgbm_scores_sample: `draws` classes for every row from the random numbers `uniform` (row_size x draws
 * doubles), under the same limits for all rows.  classes, logs and all_logs (the last two or NULL): row_size x draws. */
int tgbm_predict_sample(int row_size, float *val, int *row_ptr, int *col_ptr, Tree **model, int n_trees, int trees_per_iter, float learning_rate,
                        const TgbmTopRules *rules, int draws, const double *uniform, float temperature, int top_k, float top_p, float min_p, int *classes,
                        float *logs, float *all_logs);
int tgbm_predict_sample_dense(int row_size, int n_cols, void *x, int is_f64, Tree **model, int n_trees, int trees_per_iter, float learning_rate,
                              const TgbmTopRules *rules, int draws, const double *uniform, float temperature, int top_k, float top_p, float min_p,
                              int *classes, float *logs, float *all_logs);

#ifdef __cplusplus
}
#endif
#endif
