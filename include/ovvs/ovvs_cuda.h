#pragma once

/* B200 extensions to the ovvs C ABI.
 *
 * None of these entry points has a counterpart in the reference (its ABI is single-process,
 * host-pointer only). They exist for two kinds of caller:
 *   - callers whose queries and results already live in GPU memory (device-pointer search), and
 *   - one-process-per-GPU deployments that shard the database rows across GPUs and merge the
 *     per-shard candidates with an NCCL all-gather.
 * Everything here uses the same handles and status codes as ovvs.h. */

#include "ovvs.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- streams and errors ------------------------------------------------------------------ */

/* The cudaStream_t (as void*) that this Resources enqueues its work on. Created on first use. */
OVVS_API ovvsStatus ovvsResourcesStream(ovvsResources_t res, void** stream);

/* Waits for all work enqueued through this Resources and reports what the kernels recorded:
   OVVS_STATUS_ERROR if a kernel's bounded wait gave up (its watchdog), or a CUDA error. */
OVVS_API ovvsStatus ovvsResourcesSynchronize(ovvsResources_t res);

/* CUDA device ordinal this Resources is bound to. */
OVVS_API ovvsStatus ovvsResourcesDevice(ovvsResources_t res, int32_t* device);

/* Per-phase device timing. When enabled, each search records CUDA events on the Resources'
   stream at its phase boundaries; ovvsResourcesLastPhaseMs waits for the last search and writes
   up to `count` durations in milliseconds: [0] query preparation (+ allow bits), [1] fused
   distance / top-k kernel, [2] candidate merge + exact re-rank, [3] cross-shard all-gather and
   merge (0 on one GPU). After a k-means fit the phases are the fit's: [0] dataset upload and
   seeding, [1] the Lloyd iterations, [2] centroid download, [3] 0. After ovvsGemm / ovvsGemmEx /
   ovvsPairwiseDistance: [0] the uploads before the first output block's kernels, [1] those
   kernels (the whole call when the output fits one block, 1 GiB), [2] the rest (downloads and
   any further blocks), [3] 0. */
OVVS_API ovvsStatus ovvsResourcesSetProfiling(ovvsResources_t res, int32_t enable);
OVVS_API ovvsStatus ovvsResourcesLastPhaseMs(ovvsResources_t res, float* ms, int32_t count);

/* The same four phase durations for each of the last searches run while profiling was enabled (up
   to 64, oldest first), so back-to-back searches can be timed without synchronising after each:
   waits for the most recent one, writes min(recorded, max_searches) rows of 4 floats (ms) to `ms`
   and their number to *count, then clears the record (enabling profiling also clears it). Not in
   the reference. */
OVVS_API ovvsStatus ovvsResourcesPhaseHistoryMs(ovvsResources_t res, float* ms,
                                                int32_t max_searches, int32_t* count);

/* ---- kernel watchdog ---------------------------------------------------------------------- */

/* Every wait inside this library's kernels (on a copy, an MMA, another warp or another GPU) is
   bounded in time. A wait that runs out writes a watchdog code into the Resources' error word and
   the kernel unwinds and returns, so the device context stays usable; the next synchronising call
   on the Resources (a search, ovvsResourcesSynchronize) then returns OVVS_STATUS_ERROR. This call
   writes the code that call saw (0 if none) and clears it. Codes: 0x101-0x109 waits of the fused
   kernel (query tile, ring slot empty/full, TMEM buffer empty/full, query tile empty, unwinding,
   side slot empty/full), 0x201 the self test below. Not in the reference. */
OVVS_API ovvsStatus ovvsResourcesLastKernelError(ovvsResources_t res, int32_t* code);

/* 1 when sharded searches on this Resources share each query's bound with the other ranks: the
   fused kernel of every rank min-writes its current k-th best key for a query into every
   rank's bound array (mapped over NVLink from a CUDA virtual-memory allocation each rank
   exports to its peers), so each rank filters with the best bound found on any rank. 0 before
   the first sharded search, when peer memory cannot be shared, for cosine and large-k searches
   (which keep their bound on their own rank), or when OVVS_PEER_BOUNDS=0 is set (on every
   rank). Results are the same either way. Not in the reference. */
OVVS_API ovvsStatus ovvsResourcesPeerBounds(ovvsResources_t res, int32_t* active);

/* Runs a one-block kernel whose bounded wait is never satisfied, with a limit of `limit_ns`
   nanoseconds (1e6..5e9), and checks that the watchdog fired: the kernel returns, the
   synchronising call reports OVVS_STATUS_ERROR and the code is 0x201. Returns
   OVVS_STATUS_SUCCESS and *code = 0x201 when that is what happened. Not in the reference. */
OVVS_API ovvsStatus ovvsWatchdogSelfTest(ovvsResources_t res, int64_t limit_ns, int32_t* code);

/* ---- device-pointer search ---------------------------------------------------------------- */

/* Same contract as ovvsBruteForceSearch, but queries, bitset, neighbors and distances are device
   pointers on the Resources' device, and the call only enqueues work on the Resources' stream
   (no host synchronisation), except for k above the register lists (k beyond 28), where it waits
   for its own work once per pass to check the candidate buffers for overflow. Output rows have
   stride min(k, n). Call ovvsResourcesSynchronize
   (or synchronise the stream) before reading the results. On a sharded Resources the call is
   collective: every rank passes the same queries and receives the global result. */
OVVS_API ovvsStatus ovvsBruteForceSearchDevice(ovvsResources_t res, ovvsBruteForceIndex_t index,
                                               const float* d_queries, int64_t nq, int64_t k,
                                               const uint8_t* d_bitset, int64_t* d_neighbors,
                                               float* d_distances);

/* Same search as ovvsBruteForceSearchDevice for callers that cannot let a library allocate GPU
   memory -- e.g. a process whose free device memory is already reserved by another allocator
   (a framework's caching pool), or a latency-critical request loop where cudaMalloc/cudaFree and
   their implicit device synchronisation are not acceptable. This entry point has no counterpart
   in the reference. It allocates nothing: all intermediate buffers come from a fixed 32 MiB
   device array built into the library, which lives until the process exits. The runtime creates
   the array on a device when it loads that part of the library there; with CUDA's default lazy
   module loading this is the first call on the device, which also looks up the array's address
   (the one-time set-up). So make that first call at start-up, before another allocator takes the
   device's free memory (or set CUDA_MODULE_LOADING=EAGER). Work runs on
   `stream` (NULL = the default stream) and the call returns after it has finished. Sizes whose
   buffers do not fit the array (about 4*dim + 16 + 8*list bytes per query, list = k plus a small
   margin rounded up to 4/8/12/16/32: some 50k queries of dim 128 at k = 10) are rejected with
   OVVS_STATUS_SHAPE_MISMATCH;
   sharded indexes and k above the register-list limit return OVVS_STATUS_UNSUPPORTED. All calls on
   a device share the array and keep the last call's contents; the library clears what must start
   empty and serialises its own calls per device, because calls whose GPU work overlapped on the
   same array would race. */
OVVS_API ovvsStatus ovvsBruteForceSearchDeviceNoAlloc(ovvsResources_t res,
                                                      ovvsBruteForceIndex_t index,
                                                      const float* d_queries, int64_t nq,
                                                      int64_t k, const uint8_t* d_bitset,
                                                      int64_t* d_neighbors, float* d_distances,
                                                      void* stream);

/* Device-pointer IVF-Flat search: the contract of ovvsIvfFlatSearch (reference
   src/neighbors/indexes.cpp:302-358; outputs [nq x k], -1 / +inf past a query's candidates) with
   queries, bitset (indexed by row id, covering the index's rows), neighbors and distances in GPU
   memory on the Resources' device. Enqueues work on the Resources' stream; synchronise before
   reading the results. With the L2 metrics and k <= 10 (the tensor-core list scan) the call also
   waits once per query block for the stream's work so far, to size the scan's work items from
   the probe counts. Not in the reference. */
OVVS_API ovvsStatus ovvsIvfFlatSearchDevice(ovvsResources_t res, ovvsIvfFlatIndex_t index,
                                            const float* d_queries, int64_t nq, int64_t k,
                                            int32_t nprobe, const uint8_t* d_bitset,
                                            int64_t* d_neighbors, float* d_distances);

/* ---- rows of scores in GPU memory: drawing, routing, grouping --------------------------------- */

/* The drawn and the trained counterparts of ovvsTopk, for scores that are already on the GPU: a
   search's scores, a router's or a language model's logits. All pointers are device pointers on
   the Resources' device, aligned to their element; sizes have to be positive (rows or tokens up to
   134,217,712). An output lies neither where another does nor where an input does, but for the
   gradient that is written over its logits. Each call checks
   its arguments (INVALID_ARGUMENT, or SHAPE_MISMATCH where a size is beyond a limit), enqueues
   its kernels on `stream` (NULL = the default stream) and returns; it uses no workspace and takes
   no lock, so calls may run at once and may be captured into CUDA graphs. The caller's current
   device is left as it was. Not in the reference.

   Order: larger scores first, equal ones (-0 equals +0) by lower column, as ovvsTopk with
   `largest`. A score of -inf, and a NaN, is masked: never drawn, never chosen, no weight and no
   gradient. Any other value, the type's lowest included, is an ordinary score; where a row holds
   +inf, its softmax is shared by the columns that hold it. */

typedef enum ovvsScoreType {
  OVVS_SCORE_F32 = 0,
  OVVS_SCORE_F16 = 1,
  OVVS_SCORE_BF16 = 16
} ovvsScoreType;

/* Draws `draws` columns, with replacement, from each row of logits [rows x cols] (row stride
   `ld` >= cols elements). With weights w_j = exp((x_j - max) / temperature) and the columns of a
   row in order, the columns kept are the shortest of
     top_k   the first top_k (off: top_k <= 0),
     top_p   the fewest first columns whose weights reach top_p times the weight of the columns
             that top_k keeps (off: top_p >= 1 or NaN; at least one column),
     min_p   the columns with x_j >= max + temperature * ln(min_p), min_p at most 1 (off:
             min_p <= 0 or NaN).
   The draw for a uniform u in [0, 1) is the first column, by column number, at which the running
   sum of kept weights is above u times their total (u outside [0, 1), or NaN, counts as the
   nearest value inside, NaN as 0). A temperature that is not above 0 takes the first column in
   order with probability 1. A row with every score masked gives id -1, probability 0, kept 0.
   Weights and their sums are 64-bit integers, so that no sum rounds: a weight is a multiple of
   2^-50 of the row's largest up to 4,096 columns, of 2^-45 at 131,072 (one bit fewer for every
   doubling), less than one such step from its exponential, and one that rounds to 0 is kept like
   the others but never drawn, not for u = 0 either. (u times the total, and top_p times the
   weight, are rounded to 53 bits.)
   d_temperature, d_top_k, d_top_p, d_min_p: [rows], each may be NULL (1, off, off, off).
   d_uniforms [rows x draws]. d_ids [rows x draws]; d_probs [rows x draws] (may be NULL) gets the
   weight of each drawn column over the total that was drawn from; d_kept [rows] (may be NULL)
   the number of columns kept. cols up to 2^31 - 1. */
OVVS_API ovvsStatus ovvsSampleRowsDevice(ovvsResources_t res, const void* d_logits, int32_t type,
                                         int64_t rows, int64_t cols, int64_t ld,
                                         const float* d_temperature, const int32_t* d_top_k,
                                         const float* d_top_p, const float* d_min_p,
                                         const float* d_uniforms, int64_t draws, int64_t* d_ids,
                                         float* d_probs, int32_t* d_kept, void* stream);

typedef enum ovvsRouteScore { OVVS_ROUTE_SOFTMAX = 0, OVVS_ROUTE_SIGMOID = 1 } ovvsRouteScore;

/* A group's value: its best choice value, or the sum of its two best. */
typedef enum ovvsRouteGroupRule {
  OVVS_ROUTE_GROUP_MAX = 0,
  OVVS_ROUTE_GROUP_TOP2 = 1
} ovvsRouteGroupRule;

/* Chooses k experts for every token from logits [tokens x experts] (row stride `ld`). The scores
   s are the row's softmax or sigmoids. Experts are ordered by their logits without a bias, by
   s + bias (in 64 bits) with one. With groups > 1 the experts form `groups` groups of
   neighbours, of which the topk_groups with the best value stand (TOP2 sums s without a bias,
   s + bias with one; a group with one expert left has that one's value). d_ids [tokens x k]
   holds the chosen experts in order, -1 where none is left; d_weights [tokens x k] scale * s, or
   with `renormalize` scale * s / (sum of the chosen s), which holds also where the scores
   themselves would vanish. The bias takes no part in weights or scores. An expert whose bias is
   -inf or NaN is not chosen. d_scores [tokens x experts] (may be NULL) gets all s, 0 where
   masked. At most 1024 experts, 32 groups, k <= 32 and k <= experts (SHAPE_MISMATCH beyond). */
OVVS_API ovvsStatus ovvsRouteTopkDevice(ovvsResources_t res, const void* d_logits, int32_t type,
                                        int64_t tokens, int64_t experts, int64_t ld,
                                        const float* d_bias, int32_t score, int32_t groups,
                                        int32_t topk_groups, int32_t group_rule, int32_t k,
                                        int32_t renormalize, float scale, int32_t* d_ids,
                                        float* d_weights, float* d_scores, void* stream);

/* Gradient of ovvsRouteTopkDevice's weights, and of its scores where d_dscores is given, with
   respect to the logits, for the same logits, score, renormalize and scale and the ids it chose
   (entries outside [0, experts), and masked experts, have no part). d_dlogits [tokens x experts]
   (the logits' type, row stride `ldd`) is written whole, 0 where masked; it may be the logits'
   own memory with the same stride. The choice itself has no gradient, and neither has the bias.
   At most 1024 experts, k <= 32. */
OVVS_API ovvsStatus ovvsRouteTopkBackwardDevice(ovvsResources_t res, const void* d_logits,
                                                int32_t type, int64_t tokens, int64_t experts,
                                                int64_t ld, const int32_t* d_ids, int32_t k,
                                                int32_t score, int32_t renormalize, float scale,
                                                const float* d_dweights, const float* d_dscores,
                                                void* d_dlogits, int64_t ldd, void* stream);

/* Groups the pairs of d_ids [pairs] (a routed [tokens x k] array, flat) by expert, in pair order
   within an expert, each expert's segment padded to a multiple of `align` places. d_offsets
   [experts + 1]: the segments' starts, and the end of the last. d_order [capacity]: the pair that
   stands at each place, -1 at padding and behind the last segment; capacity has to be at least
   pairs + min(experts, pairs) * (align - 1) (SHAPE_MISMATCH below). d_position [pairs]: the place
   of each pair, -1 where its id is outside [0, experts). At most 1024 experts. */
OVVS_API ovvsStatus ovvsRoutePlanDevice(ovvsResources_t res, const int32_t* d_ids, int64_t pairs,
                                        int64_t experts, int32_t align, int32_t* d_offsets,
                                        int32_t* d_order, int64_t capacity, int32_t* d_position,
                                        void* stream);

/* ---- one process per GPU ------------------------------------------------------------------ */

/* Size in bytes of the NCCL unique id that ovvsNcclUniqueId writes (128). */
OVVS_API int32_t ovvsNcclUniqueIdSize(void);

/* Rank 0 calls this once and shares the bytes with every other rank (any transport). */
OVVS_API ovvsStatus ovvsNcclUniqueId(uint8_t* id, int32_t len);

/* Creates a Resources bound to CUDA device `device` that is rank `rank` of `world` ranks. With
   world > 1 it owns an NCCL communicator built from `nccl_id` (collective: all ranks must call).
   Searches and k-means fits through it are collective over the ranks. */
OVVS_API ovvsStatus ovvsResourcesCreateSharded(ovvsResources_t* res, int32_t device,
                                               int32_t rank, int32_t world,
                                               const uint8_t* nccl_id, int32_t len);

/* Builds this rank's shard: `n_local` rows that are rows [row_offset, row_offset + n_local) of
   the global dataset. Search results report global row ids, and a search bitset is indexed by
   global row id. */
OVVS_API ovvsStatus ovvsBruteForceBuildShard(ovvsResources_t res, const void* dataset,
                                             int64_t n_local, int64_t dim, ovvsMetric metric,
                                             ovvsDType dtype, int64_t row_offset,
                                             ovvsBruteForceIndex_t* index);

/* Collective k-means over row shards: rank r passes rows [row_offset, row_offset + n_local) of a
   dataset with n_total rows. Seeding picks the same global rows as ovvsKMeansFit would on the
   whole dataset; per-iteration sums and counts are all-reduced, so every rank ends with the same
   centroids. */
OVVS_API ovvsStatus ovvsKMeansFitShard(ovvsResources_t res, const float* dataset, int64_t n_local,
                                       int64_t row_offset, int64_t n_total, int64_t dim,
                                       int32_t nclusters, int32_t iters,
                                       ovvsKMeansModel_t* model);

#ifdef __cplusplus
}
#endif
