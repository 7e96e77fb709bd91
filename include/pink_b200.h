/*
 * pink_b200.h -- C ABI of the B200-native implementation of PINK's
 * rotation/flip-invariant SOM hot path (rotate/flip -> distance matrix ->
 * minimum over rotations -> best matching unit -> neighbourhood update, and
 * the mapping variant).
 *
 * The reference has no FFI layer for this path: its boundary is the C++
 * template specialisation Trainer<..., UseGPU=true> / Mapper<..., UseGPU=true>
 * (src/SelfOrganizingMapLib/Trainer.h:198-333, Mapper.h:126-229), which owns
 * device buffers and calls three CudaLib entry points that take
 * thrust::device_vector arguments.  The functions below are what a binding of
 * that boundary needs: plain pointers and sizes, an opaque context in place of
 * the Trainer/Mapper object's device state, and an int status in place of
 * exceptions and exit().  Each entry names the reference code it stands for.
 *
 * Conventions
 *   - every function returns PINK_B200_OK (0) or a negative PINK_B200_E* code;
 *     nothing throws, nothing calls exit().  pink_b200_last_error() returns a
 *     message for the calling thread's most recent failure.
 *   - "host" pointers are ordinary (pageable or pinned) host memory, "dev"
 *     pointers are device memory of the context's device.
 *   - images are float32 [C][id][id] (C == 1 for 2-D data), SOMs are float32
 *     [N][C][nd][nd], both row-major without padding.
 *   - a context is used from one host thread at a time.
 *   - there is no CPU fallback: every compute entry runs CUDA kernels and
 *     fails with PINK_B200_ECUDA where no sm_100 device is present.
 */
#ifndef PINK_B200_H
#define PINK_B200_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define PINK_B200_OK          0
#define PINK_B200_EINVAL     -1   /* bad argument or unsupported configuration      */
#define PINK_B200_ECUDA      -2   /* CUDA runtime / driver error                    */
#define PINK_B200_ENCCL      -3   /* NCCL error or NCCL library not loadable        */
#define PINK_B200_ETIMEOUT   -4   /* a bounded device-side wait expired             */
#define PINK_B200_ESTATE     -5   /* call not valid in the context's current state  */

/* Distance modes; numbering of pink::DataType (src/UtilitiesLib/DataType.h:17-22). */
#define PINK_B200_FLOAT   0
#define PINK_B200_UINT16  1
#define PINK_B200_UINT8   2

/* Shape of the distance region (src/UtilitiesLib/EuclideanDistanceShape.h:15-19). */
#define PINK_B200_QUADRATIC 0
#define PINK_B200_CIRCULAR  1

/* Interpolation (src/UtilitiesLib/Interpolation.h:15-19); only BILINEAR exists
 * on the reference's GPU path (src/CudaLib/generate_rotated_images.h:119-121). */
#define PINK_B200_NEAREST_NEIGHBOR 0
#define PINK_B200_BILINEAR         1

/* SOM grid layouts (src/UtilitiesLib/Layout.h:15-19). */
#define PINK_B200_LAYOUT_CARTESIAN 0
#define PINK_B200_LAYOUT_HEXAGONAL 1

/* Neighbourhood functions (src/UtilitiesLib/DistributionFunctor.h:32-104). */
#define PINK_B200_FUNC_GAUSSIAN        0   /* p0 = sigma, p1 = damping */
#define PINK_B200_FUNC_UNITY_GAUSSIAN  1   /* p0 = sigma, p1 = damping */
#define PINK_B200_FUNC_MEXICAN_HAT     2   /* p0 = sigma, p1 = damping */
#define PINK_B200_FUNC_STEP            3   /* p0 = value               */

typedef struct pink_b200_ctx pink_b200_ctx;

/* Everything the Trainer / Mapper constructors take that shapes device state
 * (src/SelfOrganizingMapLib/Trainer.h:211-215, Mapper.h:134-137). */
typedef struct pink_b200_config {
    uint32_t n_neurons;        /* N: neurons of the whole SOM                                  */
    uint32_t channels;         /* C: 1 for 2-D images, dimension 0 of 3-D images ("spacing")   */
    uint32_t image_dim;        /* id: images are square                                        */
    uint32_t neuron_dim;       /* nd                                                           */
    uint32_t ed_dim;           /* euclidean_distance_dim                                       */
    uint32_t ed_shape;         /* PINK_B200_QUADRATIC                                          */
    uint32_t n_rotations;      /* number_of_rotations: 1 or a multiple of 4                    */
    uint32_t use_flip;         /* 0 / 1                                                        */
    uint32_t dist_type;        /* PINK_B200_FLOAT / UINT16 / UINT8                             */
    uint32_t interpolation;    /* PINK_B200_BILINEAR                                           */
    int32_t  device;           /* CUDA device ordinal                                          */
    uint32_t rank;             /* this process's index among the neuron shards                 */
    uint32_t world_size;       /* number of neuron shards (1 = whole SOM on this device)       */
    uint32_t max_batch;        /* images staged per internal batch (0 = default)               */
} pink_b200_config;

/* Message of the calling thread's most recent failing call ("" if none). */
const char* pink_b200_last_error(void);

/* Library version string. */
const char* pink_b200_version(void);

/* ---- context life cycle ---------------------------------------------------- */

/* Validates the configuration (errors of TrainerCommon / MapperCommon,
 * src/SelfOrganizingMapLib/Trainer.h:66-67, Mapper.h:59-66, and "Images must
 * be quadratic" is implied by image_dim) and allocates the device state the
 * reference allocates in the Trainer / Mapper constructors
 * (Trainer.h:216-260, Mapper.h:138-178), including the cos/sin tables. */
int pink_b200_create(const pink_b200_config* cfg, pink_b200_ctx** out);
int pink_b200_destroy(pink_b200_ctx* ctx);

/* The neurons that live on this context's device: global neurons first + j * stride, j < count, with
 * stride = pink_b200_shard_stride(ctx).  count is N/world (+1 for the first N % world ranks), the sizes of
 * the reference's multi-GPU split (src/CudaLib/generate_euclidean_distance_matrix_first_step_multi_gpu.h:65-77).
 * By default the shards are interleaved (first = rank, stride = world_size), so that the neurons around any best
 * matching unit -- the ones an image rewrites -- are spread evenly over the ranks; option "sharding" = 1 selects
 * the reference's contiguous ranges (stride 1).  Mapping results are in this local order. */
int pink_b200_shard(const pink_b200_ctx* ctx, uint32_t* first, uint32_t* count);
uint32_t pink_b200_shard_stride(const pink_b200_ctx* ctx);
/* The reference's contiguous split as a pure host function (no context, no GPU). */
int pink_b200_shard_range(uint32_t n_neurons, uint32_t world_size, uint32_t rank, uint32_t* first, uint32_t* count);

/* Switches of a context, to be set after pink_b200_create and before pink_b200_comm_init /
 * pink_b200_set_som (no reference counterpart: the reference has one fixed launch sequence).  Unknown
 * names and values out of range return PINK_B200_EINVAL.
 *   "step_kernel"          0 (default) whole batches of training steps in one persistent kernel where the
 *                          geometry allows it; 1 two kernels per image (distance, update); 2 four kernels
 *                          per image (distance, best matching unit, work list, update)
 *   "sharding"             0 (default) interleaved neuron shards, 1 contiguous ranges as in the reference
 *   "exchange"             0 (default) per-rank records through peer memory where possible; 1 NCCL all-gather
 *   "rotation_sharing"     -1 (default) pairs of ranks share the rotation work; 0 every rank rotates every
 *                          image; g >= 2 groups of g consecutive ranks share
 *   "rotation_overlap"     1 puts the rotation kernels on a second, low-priority stream (default 0)
 *   "mma_pairs"            0 keeps the distance kernel from pairing blocks (default 1)
 *   "f32_filter"           0 computes float32 distances with the all-pairs exact kernel instead of the tensor-core
 *                          estimate + exact pass (default 1)
 *   "cooperative_launch"   0 launches the persistent kernel without the cooperative attribute (default 1).  Its
 *                          blocks wait for one another, so this is only for a device with nothing else running,
 *                          under a profiler that refuses cooperative launches; a block that is not resident
 *                          ends the batch with PINK_B200_ETIMEOUT instead of a hang
 *   "exchange_timeout_ms"  wall-clock limit of every device-side wait for another rank (default 20000).  The
 *                          ranks must enqueue each batch of steps within this time of one another. */
int pink_b200_set_option(pink_b200_ctx* ctx, const char* name, long long value);

/* ---- multi-GPU: one process per GPU, neuron shards, NCCL for the BMU exchange
 * (replaces the per-image cudaMemcpyPeer traffic of
 *  src/CudaLib/generate_euclidean_distance_matrix_first_step_multi_gpu.h:87-104,184-193). */

/* Rank 0 fills a 128-byte NCCL unique id; the caller distributes it. */
int pink_b200_comm_unique_id(void* id128);
/* Collective over all ranks of the job; required before training when world_size > 1. */
int pink_b200_comm_init(pink_b200_ctx* ctx, const void* id128);

/* ---- SOM and neighbourhood table ------------------------------------------- */

/* Upload the SOM (host, [N][P] float, the WHOLE map: each rank keeps its
 * shard) and build the distance operand.  Stands for the device copy taken at
 * construction, Trainer.h:219 / Mapper.h:140. */
int pink_b200_set_som(pink_b200_ctx* ctx, const float* host_som);
/* Write this rank's shard into its rows (first + j * stride) of host_som ([N][P]);
 * other rows are left untouched.  Stands for Trainer::update_som(), Trainer.h:306-309. */
int pink_b200_get_som(pink_b200_ctx* ctx, float* host_som);
/* Upload the N x N update-factor table F[bmu * N + n] the reference builds on
 * the host from the layout distance and the distribution function
 * (Trainer.h:69-76, uploaded at :243).  Each rank keeps its columns. */
int pink_b200_set_update_factors(pink_b200_ctx* ctx, const float* host_factors);

/* Host helpers (no GPU involved) for the tables the reference computes on the
 * host.  Number of neurons of a SOM grid: dim0 * dim1 (cartesian) or the
 * row-packed hexagon of side dim0 (HexagonalLayout.h:61-64). */
uint32_t pink_b200_som_size(uint32_t som_layout, uint32_t dim0, uint32_t dim1);
/* out[i * N + j] = layout.get_distance(i, j) (CartesianLayout.h:47-60,108-114;
 * HexagonalLayout.h:90-118). */
int pink_b200_som_distances(uint32_t som_layout, uint32_t dim0, uint32_t dim1, float* out);
/* out[i * N + j] = func(distance) if max_update_distance <= 0 or distance <
 * max_update_distance, else 0 -- the TrainerCommon loop (Trainer.h:69-76) for
 * the built-in functors (DistributionFunctor.cpp:18-59).  Callers with their
 * own distribution function fill the table themselves. */
int pink_b200_update_factors(uint32_t som_layout, uint32_t dim0, uint32_t dim1, uint32_t func, float p0, float p1,
                             float max_update_distance, float* out);

/* The same without an N x N table (no reference counterpart; the reference evaluates its distribution function N^2
 * times and keeps N^2 floats, Trainer.h:69-76 -- 7.8 million calls and 31 MB for 2,791 neurons).  The map distance of
 * two neurons takes few distinct values: it depends only on the absolute coordinate differences (cartesian grids of
 * up to three dimensions; dim2 = 1 for two) or is the hop count (hexagonal; dim2 = 1).  pink_b200_distance_classes
 * returns their number and (if `distances` is not NULL) the distance of every class; a caller with its own
 * distribution function evaluates it once per class, applies the max_update_distance cut-off and hands the result to
 * pink_b200_set_update_lut.  pink_b200_update_lut does that for the built-in functors, pink_b200_set_update_function
 * both steps.  The factors are identical to the table's, bit for bit.  pink_b200_som_coordinates: the grid
 * position (x, y, z, 0 -- hexagonal: axial q, r) of every neuron as int16[N][4]. */
uint32_t pink_b200_distance_classes(uint32_t som_layout, uint32_t dim0, uint32_t dim1, uint32_t dim2, float* distances,
                                    uint32_t capacity);
int pink_b200_som_coordinates(uint32_t som_layout, uint32_t dim0, uint32_t dim1, uint32_t dim2, int16_t* out);
int pink_b200_update_lut(uint32_t som_layout, uint32_t dim0, uint32_t dim1, uint32_t dim2, uint32_t func, float p0, float p1,
                         float max_update_distance, float* lut, uint32_t capacity);
int pink_b200_set_update_lut(pink_b200_ctx* ctx, uint32_t som_layout, uint32_t dim0, uint32_t dim1, uint32_t dim2,
                             const float* host_lut, uint32_t n_classes);
int pink_b200_set_update_function(pink_b200_ctx* ctx, uint32_t som_layout, uint32_t dim0, uint32_t dim1, uint32_t dim2,
                                  uint32_t func, float p0, float p1, float max_update_distance);

/* The same two tables for a three-dimensional cartesian SOM of dim0 x dim1 x dim2
 * neurons (CartesianLayout<3>, CartesianLayout.h:116-123 for the position of an
 * array index; the command line tool's --som-depth > 1, main_gpu.cu:24-25). */
int pink_b200_som_distances_3d(uint32_t dim0, uint32_t dim1, uint32_t dim2, float* out);
int pink_b200_update_factors_3d(uint32_t dim0, uint32_t dim1, uint32_t dim2, uint32_t func, float p0, float p1,
                                float max_update_distance, float* out);

/* ---- training --------------------------------------------------------------
 * n sequential training steps; image i+1 sees the SOM updated by image i.
 * Stands for n calls of Trainer<...,true>::operator() (Trainer.h:263-304).
 * Asynchronous with respect to the host except for staging of host images;
 * results are observed through get_som / get_update_counts / synchronize. */
int pink_b200_train(pink_b200_ctx* ctx, const float* host_images, uint64_t n);
int pink_b200_train_device(pink_b200_ctx* ctx, const float* dev_images, uint64_t n);
/* Per-neuron BMU hit counters, [N] (all ranks hold the same totals only for
 * their own shard; other entries are zero).  Stands for get_update_info(),
 * Trainer.h:79, counted at :302-303. */
int pink_b200_get_update_counts(pink_b200_ctx* ctx, uint32_t* host_counts);
/* Optional: global BMU index of each of the last train call's images (host, [n]);
 * only the rank owning the BMU writes an entry, others read 0xFFFFFFFF. */
int pink_b200_get_bmu_log(pink_b200_ctx* ctx, uint32_t* host_bmus, uint64_t n);

/* ---- mapping ---------------------------------------------------------------
 * For each of n images: dist[i][j] = sqrt(min over transforms of the scaled
 * squared distance to local neuron j), rot[i][j] = the first transform
 * attaining it; j runs over this rank's shard (count entries per image).
 * Stands for n calls of Mapper<...,true>::operator() (Mapper.h:181-208). */
int pink_b200_map(pink_b200_ctx* ctx, const float* host_images, uint64_t n, float* host_dist, uint32_t* host_rot);
int pink_b200_map_device(pink_b200_ctx* ctx, const float* dev_images, uint64_t n, float* dev_dist, uint32_t* dev_rot);

/* ---- mapping with routes and a read-out (no reference counterpart) ------------
 * pink_b200_map, followed on the device by the read-out operators (see "read-out of a map" below): the neurons that speak for
 * every image, and what a table of values per neuron -- labels, redshifts, prototypes -- says about it. */
typedef struct pink_b200_route_config pink_b200_route_config;      /* defined below */

/* Table of `dims` float32 values per neuron ([N][dims], host; NULL removes it).  dense = 0: an image's result is the sum of its routed
 * neurons' values, in float32.  dense = 1: of ALL neurons' values with their scores as weights, a product on the tensor cores into
 * which scores and values enter rounded to bfloat16 (as does its result): for many values of which two digits are wanted.  The values of a
 * neuron that the mapping call masks do not enter it, be they infinite or NaN; those of a neuron whose score is zero otherwise do. */
int pink_b200_set_values(pink_b200_ctx* ctx, const float* host_values, uint32_t dims, uint32_t dense);

/* Results of pink_b200_map_routes (host pointers; each may be NULL). */
typedef struct pink_b200_route_results {
    float* dist;               /* [n][N] distances and ...                                                              */
    uint32_t* rot;             /* [n][N] ... transforms, as pink_b200_map returns them                                  */
    uint32_t* neurons;         /* [n][top_k] chosen neurons, 0xFFFFFFFF where there is none                             */
    float* weights;            /* [n][top_k] their weights                                                              */
    uint32_t* rotations;       /* [n][top_k] the transforms in which the image meets them, 0xFFFFFFFF where there is none */
    float* out;                /* [n][dims] read-out of the table of pink_b200_set_values                               */
} pink_b200_route_results;

/* Maps n images and routes each by its distances: cfg as for pink_b200_op_route (n_neurons = N; slope negative, so that near neurons are
 * preferred), host_bias ([N], nullable) and host_mask ([N] bytes, nullable) alike.  For contexts that hold the whole map
 * (world_size == 1).  Copies back what is asked for: top_k routes an image instead of N distances. */
int pink_b200_map_routes(pink_b200_ctx* ctx, const pink_b200_route_config* cfg, const float* host_images, uint64_t n, const float* host_bias,
                         const uint8_t* host_mask, const pink_b200_route_results* results);

/* Wait for all queued work of the context; surfaces asynchronous errors and
 * device-side time-outs. */
int pink_b200_synchronize(pink_b200_ctx* ctx);

/* The CUDA stream (cudaStream_t) the context launches on, for callers that
 * time or order work against it. */
void* pink_b200_stream(pink_b200_ctx* ctx);

/* Number of CUDA kernels the context has launched since it was created (the
 * reference has no counterpart; benchmarks report it). */
uint64_t pink_b200_launch_count(pink_b200_ctx* ctx);

/* How the ranks exchange their best-matching-unit records every step (no
 * reference counterpart: the reference trains on one GPU).  PEER: each rank
 * stores its record into every rank's memory over NVLink and the update kernel
 * waits for them (ranks on one node, one GPU each); PEER_SHARED_ROTATION: the
 * same, and the ranks also share the rotation work -- each computes the rotation
 * sets of its part of every batch of images and copies them into all ranks'
 * buffers; NCCL: an all-gather per step; NONE: a single rank or no communicator yet. */
enum { PINK_B200_EXCHANGE_NONE = 0, PINK_B200_EXCHANGE_NCCL = 1, PINK_B200_EXCHANGE_PEER = 2,
       PINK_B200_EXCHANGE_PEER_SHARED_ROTATION = 3 };
int pink_b200_exchange_kind(pink_b200_ctx* ctx);

/* Totals over all training steps of this context (this rank's shard): out[0] =
 * neurons that had a non-zero update factor, out[1] = neurons written back.
 * The reference rewrites every neuron (update_neurons.h:34-49); here a neuron
 * whose new values all equal the old ones bit for bit is read but not written. */
int pink_b200_get_update_stats(pink_b200_ctx* ctx, uint64_t* out);

/* Opt-in phase timing (the reference only has a wall clock around the whole
 * run, src/Pink/main.cpp:37-62).  After profile_begin, CUDA events on the
 * context's streams bracket the kernels of each of the next max_steps
 * training steps; profile_end waits for them and returns the summed device
 * time in milliseconds of {rotation sets (batched, overlapped with the steps),
 * distance, BMU + exchange, update} and the number of steps covered.  Event records perturb the pipeline slightly:
 * use it to apportion time between kernels, not to measure throughput. */
int pink_b200_profile_begin(pink_b200_ctx* ctx, uint32_t max_steps);
int pink_b200_profile_end(pink_b200_ctx* ctx, double ms_sum[4], uint64_t* steps);
/* After profile_end, for a context that trains with the persistent kernel (all zeros otherwise):
 * out[0] = mean device time of one launch in microseconds (CUDA events), out[1] = mean images per launch,
 * out[2..6] = mean microseconds per image, read from device-timer stamps of block 0, of: its own distance
 * tiles (TMA + MMA + epilogue), waiting for the other blocks at the first grid barrier, best matching unit
 * (+ exchange between ranks) and work list, rewriting its own neurons, waiting at the second grid barrier;
 * out[7] unused. */
int pink_b200_profile_detail(pink_b200_ctx* ctx, double out[8]);
/* The raw stamps behind it, [steps][blocks][12] words: nanoseconds of the device timer when (0) the image began,
 * (1) the block had reduced its own distance tiles, (2) it had passed the first grid barrier, (3) its work
 * list was built, (4) its own neurons were rewritten and stored, (5) it had passed the second grid barrier;
 * (6) neuron planes it rewrote, (7) distance tiles it computed; inside the phases: (8) first operand slice
 * arrived, (9) last MMA issued, (10) accumulators complete, (11) first neuron plane arrived.  *blocks and
 * *steps are always set; `out` may be NULL to ask for the sizes only. */
int pink_b200_profile_stamps(pink_b200_ctx* ctx, uint64_t* out, uint64_t capacity, uint32_t* blocks, uint64_t* steps);

/* float32 distances (mapping and training) run as an estimate of all N x T distances on the tensor cores followed
 * by exact sums for the transforms the estimate cannot rule out (option "f32_filter" = 0 computes all of them exactly instead; the
 * results are the same up to the summation order of the exact sums).  out[0] = pairs estimated so far,
 * out[1] = exact sums formed, out[2] = largest |estimate - exact| / (|a|^2 + |b|^2) seen among those,
 * out[3] = the error bound the selection assumes for that ratio. */
int pink_b200_map_filter_stats(pink_b200_ctx* ctx, double out[4]);

/* Ceiling of the integer tensor pipe as the distance kernels drive it: tera-operations per second of
 * tcgen05.mma kind::i8 (128 rows x n columns per CTA; pair != 0: CTA pairs, 256 x n per instruction) issued
 * back to back on operands already in shared memory, one CTA (pair) per SM.  n: multiple of 16, 16..256.
 * A measuring aid: the distance kernels' rates are quoted against it. */
int pink_b200_mma_i8_peak(int device, uint32_t n, int pair, double* tops);

/* ---- one process, several GPUs ------------------------------------------------
 * The reference's Trainer / Mapper use every visible GPU of the process on their own
 * (src/CudaLib/CudaLib.cu:56-76; neurons split over the GPUs with a host thread per extra GPU,
 * src/CudaLib/generate_euclidean_distance_matrix_first_step_multi_gpu.h:47-196).  A group is that for this
 * library: it owns one context per device and drives them from host threads of its own.
 *   training: the neurons are sharded over the devices (rank r on devices[r]) and the shards' records are
 *             exchanged through peer memory, as between processes;
 *   mapping:  every device holds the whole map and the images of a call are dealt to the devices in contiguous
 *             ranges; results are in the order of the images.  No communication.
 * `devices` lists CUDA ordinals; NULL takes the visible sm_100 devices (at most n_devices of them when n_devices
 * is not 0).  cfg->device, rank and world_size are ignored.  SOM, factors, counters and results are those of
 * the WHOLE map: a caller never sees the shards. */
typedef struct pink_b200_group pink_b200_group;
int pink_b200_device_count(void);                  /* visible sm_100 devices */
int pink_b200_group_create(const pink_b200_config* cfg, const int32_t* devices, uint32_t n_devices, pink_b200_group** out);
int pink_b200_group_destroy(pink_b200_group* group);
uint32_t pink_b200_group_size(const pink_b200_group* group);
int pink_b200_group_set_option(pink_b200_group* group, const char* name, long long value);
int pink_b200_group_set_som(pink_b200_group* group, const float* host_som);
int pink_b200_group_get_som(pink_b200_group* group, float* host_som);
int pink_b200_group_set_update_factors(pink_b200_group* group, const float* host_factors);
int pink_b200_group_set_update_lut(pink_b200_group* group, uint32_t som_layout, uint32_t dim0, uint32_t dim1, uint32_t dim2,
                                   const float* host_lut, uint32_t n_classes);
int pink_b200_group_train(pink_b200_group* group, const float* host_images, uint64_t n);
int pink_b200_group_get_update_counts(pink_b200_group* group, uint32_t* host_counts);
int pink_b200_group_synchronize(pink_b200_group* group);
int pink_b200_group_map(pink_b200_group* group, const float* host_images, uint64_t n, float* host_dist, uint32_t* host_rot);
int pink_b200_group_set_values(pink_b200_group* group, const float* host_values, uint32_t dims, uint32_t dense);
int pink_b200_group_map_routes(pink_b200_group* group, const pink_b200_route_config* cfg, const float* host_images, uint64_t n,
                               const float* host_bias, const uint8_t* host_mask, const pink_b200_route_results* results);

/* Page-locked host memory for image and result buffers (the copies of pink_b200_train / pink_b200_map then run
 * asynchronously at full speed; pageable memory works too, slower).  The reference reads every image into
 * pageable memory (src/SelfOrganizingMapLib/DataIterator.h). */
int pink_b200_host_alloc(void** out, uint64_t bytes);
int pink_b200_host_free(void* ptr);

/* ---- single stages on device buffers (what the context calls internally) ---
 * Exposed for kernel-level parity tests and benchmarks.  `stream` is a
 * cudaStream_t (NULL = default stream).  Operand layout: integer modes use
 * rows of `row_stride` bytes (a multiple of 128, zero beyond K) per plane,
 * uint16 as two planes (high bytes, low bytes); float mode uses rows of
 * `row_stride` floats (a multiple of 32, zero beyond K). */

/* Row stride (in elements) the library uses for a distance length of K elements. */
uint32_t pink_b200_operand_stride(uint32_t K, uint32_t dist_type);

/* Rotation set of n_img images: base rotations (float, [n_img][max(R/4,1)][C][nd][nd],
 * may be NULL when shared memory holds a base) and the distance operand rows of
 * all T transforms with their sums of squares.  Stands for
 * SpatialTransformerGPU (src/CudaLib/generate_rotated_images.h:56-294) plus the
 * transform half of generate_euclidean_distance_matrix's crop/convert
 * (src/CudaLib/generate_euclidean_distance_matrix.h:86-112). */
int pink_b200_op_rotate(const pink_b200_config* cfg, const float* dev_images, uint32_t n_img,
                        float* dev_base, void* dev_b0, void* dev_b1, void* dev_bnorm, void* stream);

/* Same computation and arguments as pink_b200_op_rotate, for callers that cannot
 * allocate device memory: it calls neither cudaMalloc nor cudaFree nor any other
 * allocating routine.  (This entry has no counterpart in the reference.)
 * Who needs it: code that runs while the CUDA allocator must not be entered --
 * inside the callbacks of a caching allocator or memory pool, in a process that
 * has handed all device memory to its own arena, or in a loop that cannot afford
 * the implicit device synchronisation of cudaMalloc / cudaFree.
 * The table of rotation angles (the scratch pink_b200_op_rotate allocates per
 * call) lives in a fixed 32 KB device array inside the library, held by every GPU
 * that loads it until the process exits.  Limits and rules:
 *   - at most 16384 rotations (4096 per quadrant); more returns PINK_B200_EINVAL;
 *   - the first call on a device (and for each distance type) looks up the array's device address and
 *     loads the kernel; that first call may allocate inside the CUDA driver (module loading), so make one
 *     warm-up call per device and distance type before entering a region where allocation is forbidden;
 *     only later calls are allocation-free;
 *   - all calls share the one array (each overwrites the part it uses), so two
 *     calls whose GPU work may overlap -- different streams or host threads --
 *     race; serialise them.  The call returns after its work on `stream` is done. */
int pink_b200_op_rotate_static(const pink_b200_config* cfg, const float* dev_images, uint32_t n_img,
                               float* dev_base, void* dev_b0, void* dev_b1, void* dev_bnorm, void* stream);

/* SOM half of the crop/convert (generate_euclidean_distance_matrix.h:64-84). */
int pink_b200_op_quantize_som(const pink_b200_config* cfg, const float* dev_som, uint32_t n_neurons,
                              void* dev_a0, void* dev_a1, void* dev_anorm, void* stream);

/* Distance of every (neuron, transform) pair reduced to the per-neuron minimum
 * key (code << shift | transform; shift 32, or 16 for uint16), merged into
 * dev_keys with an unsigned minimum (fill with 0xFF bytes first).  dev_matrix
 * (nullable) receives the full [n_img][n][T] matrix: uint32 (uint8 mode),
 * uint64 (uint16), float (float).  Stands for
 * generate_euclidean_distance_matrix_first_step + _second_step
 * (src/CudaLib/generate_euclidean_distance_matrix_first_step.h:17-52,
 *  ..._second_step.h:43-62). */
int pink_b200_op_distance(uint32_t dist_type, uint32_t n_neurons, uint32_t n_transforms, uint32_t K,
                          const void* dev_a0, const void* dev_a1, const void* dev_anorm,
                          const void* dev_b0, const void* dev_b1, const void* dev_bnorm, uint32_t n_img,
                          unsigned long long* dev_keys, void* dev_matrix, void* stream);

/* Waits for the device and reports (then clears) a time-out recorded by a
 * pink_b200_op_distance, pink_b200_op_product or pink_b200_op_gated launch: PINK_B200_OK or PINK_B200_ETIMEOUT. */
int pink_b200_op_status(void);

/* ---- read-out of a map ------------------------------------------------------------
 * What comes behind the mapping (no reference counterpart; the reference stops at the distances): choosing, for every
 * image, the neurons that speak for it (route), adding up what these neurons stand for -- labels, prototypes, any table
 * with a row per neuron -- with the routes' weights (read_out), and the dense product act(x W^T + b) + r for read-outs
 * over all neurons at once, learned routers and heads (product).  Each comes with its backward pass.
 *
 * All pointers are device pointers of the CURRENT device, `stream` is a cudaStream_t of it (NULL = default stream).
 * The calls only launch kernels: they allocate nothing, copy nothing, do not synchronise, and may be captured into
 * a graph.  Where a call needs scratch memory, the caller passes it; two calls (or two graphs) that may run at the same
 * time need scratch of their own.  Outputs must not overlap inputs unless a comment says so.  Matrices are row-major;
 * a leading dimension `ld_*` is the distance from one row to the next in ELEMENTS (at least the row's length; elements
 * between the rows do not enter the results and are not written).  Results do not depend on the order in which blocks run: the same call gives
 * the same bits again.  Zero rows (n == 0) are allowed everywhere. */

/* Element types. */
#define PINK_B200_F32   0
#define PINK_B200_BF16  1
#define PINK_B200_F16   2

/* Scores of the neurons of one image. */
#define PINK_B200_SCORE_SOFTMAX 0
#define PINK_B200_SCORE_SIGMOID 1

/* Activations of pink_b200_op_product (GELU: the exact form, z * Phi(z)). */
#define PINK_B200_ACT_NONE    0
#define PINK_B200_ACT_RELU    1
#define PINK_B200_ACT_GELU    2
#define PINK_B200_ACT_SILU    3
#define PINK_B200_ACT_SIGMOID 4

#define PINK_B200_MAX_ROUTES         32      /* top_k of a route                    */
#define PINK_B200_MAX_ROUTED_NEURONS 32768   /* neurons a route can choose from     */
#define PINK_B200_MAX_ROUTE_GROUPS   256     /* groups of neurons                   */

struct pink_b200_route_config {
    uint32_t n_neurons;        /* N: 1 .. 32768                                                                 */
    uint32_t top_k;            /* k: neurons per image, 1 .. min(N, 32)                                          */
    uint32_t score;            /* PINK_B200_SCORE_SOFTMAX / SIGMOID                                              */
    uint32_t renormalise;      /* 1: the k weights of an image add up to `scale`                                 */
    uint32_t n_groups;         /* groups of N / n_groups consecutive neurons (1 = no groups); divides N, <= 256  */
    uint32_t top_groups;       /* groups an image's neurons may come from, 1 .. n_groups                         */
    uint32_t group_best;       /* value of a group: its best neuron (1) or the sum of its two best (2)           */
    float slope;               /* logit = slope * value; negative for distances                                  */
    float scale;               /* weights are multiplied by it; > 0                                              */
};

/* Routes of n images.  dev_values: [n][N] distances or learned scores of element type `type`.
 *   logit   l = slope * value, rounded to float32.  A neuron takes part if its mask (dev_mask: [N] bytes, nullable) is not
 *           zero and l is neither NaN nor -infinity; l = +infinity counts as the largest float.
 *   choice  c = l + bias (dev_bias: [N], nullable), rounded to float32: the bias shifts which neurons are chosen and does not
 *           enter the weights.  It is added to the LOGIT, a distance times the slope, and groups are compared by logits; gates that add their
 *           bias to the sigmoid or softmax score, or rank groups by sums of scores, choose otherwise under a bias or with group_best = 2.  A neuron whose c is NaN or -infinity is not chosen; +infinity counts as the largest float.
 *   groups  (n_groups > 1) the top_groups groups of the largest value stay, of equal ones the first; a group's value is its
 *           largest c, or (group_best = 2) the float32 sum of its two largest, held to the range of finite floats (one alone where it
 *           has no second).
 *   chosen  the k largest c of what stays, in descending order, of equal ones the first neuron.
 *   weight  scale * p, p = softmax of l over the neurons that take part, or sigmoid(l); renormalised: scale * p / (sum of
 *           the chosen p), formed relative to the largest of them, so that it never divides zero by zero.
 * dev_neurons: [n][k], 0xFFFFFFFF where an image has fewer than k neurons to choose from (weight 0); dev_weights: [n][k].
 * dev_load (nullable): [N] counters, to which the images' choices are ADDED.
 * dev_scores (nullable): p of every neuron, [n][ld_scores] of element type scores_type, zero where it takes no part; a p below
 * 2^-126 may be zero, and so may a weight that is not renormalised. */
int pink_b200_op_route(const pink_b200_route_config* cfg, uint64_t n, uint32_t type, const void* dev_values, uint64_t ld_values,
                       const float* dev_bias, const uint8_t* dev_mask, uint32_t* dev_neurons, float* dev_weights,
                       uint32_t* dev_load, uint32_t scores_type, void* dev_scores, uint64_t ld_scores, void* stream);

/* Gradient of a route with respect to its values, given those of its weights (dev_dweights: [n][k]; those of absent routes are
 * not read) and of its dense scores (dev_dscores, nullable: [n][ld_dscores] of element type `type`).  The choice is piecewise
 * constant and has no gradient.  dev_neurons / dev_weights: as pink_b200_op_route wrote them (entries beyond N count as
 * absent); a neuron listed twice counts twice.  dev_dvalues: [n][ld_dvalues] of element type `type`; zero where a neuron takes no part.
 * n_groups, top_groups and group_best are not looked at. */
int pink_b200_op_route_backward(const pink_b200_route_config* cfg, uint64_t n, uint32_t type, const void* dev_values, uint64_t ld_values,
                                const uint8_t* dev_mask, const uint32_t* dev_neurons, const float* dev_weights,
                                const float* dev_dweights, const void* dev_dscores, uint64_t ld_dscores, void* dev_dvalues,
                                uint64_t ld_dvalues, void* stream);

/* One step towards even loads: new_bias = bias + rate * sign(mean load - load), the mean over the neurons whose mask is not zero
 * (nullable: all); a masked neuron keeps its bias.  The comparison is exact (whole numbers).  dev_new_bias may be dev_bias. */
int pink_b200_op_route_balance(uint32_t n_neurons, const uint32_t* dev_load, const uint8_t* dev_mask, float rate, const float* dev_bias,
                               float* dev_new_bias, void* stream);

/* Read-out of routed neurons: out_i = sum over j < top_k of weights[i][j] * values[neurons[i][j]] (+ residual_i), summed in
 * float32 in the order of the routes, rounded once.  dev_values: [N][ld_values] table of `dims` elements per neuron; entries of
 * dev_neurons beyond N are left out.  values, residual (nullable) and out are of element type `type`.
 * dev_out may be dev_residual (same leading dimension). */
int pink_b200_op_read_out(uint32_t type, uint32_t n_neurons, uint32_t dims, const void* dev_values, uint64_t ld_values, uint64_t n,
                          uint32_t top_k, const uint32_t* dev_neurons, const float* dev_weights, const void* dev_residual,
                          uint64_t ld_residual, void* dev_out, uint64_t ld_out, void* stream);

/* Its backward pass: dweights[i][j] = <dout_i, values[neurons[i][j]]> (0 where absent), [n][top_k] float32, and
 * dvalues[e] = sum of weights[i][j] * dout_i over the routes to e, in a fixed order, [N][ld_dvalues] of element type
 * `type`, zero for neurons without routes.  Either may be NULL.  n_neurons <= 32768, n * top_k < 2^31.  dev_workspace: at
 * least pink_b200_read_out_workspace(...) bytes, 16-byte aligned; its content need not survive between calls (not read for dvalues == NULL). */
uint64_t pink_b200_read_out_workspace(uint32_t n_neurons, uint32_t dims, uint64_t n, uint32_t top_k);
int pink_b200_op_read_out_backward(uint32_t type, uint32_t n_neurons, uint32_t dims, const void* dev_values, uint64_t ld_values,
                                   uint64_t n, uint32_t top_k, const uint32_t* dev_neurons, const float* dev_weights,
                                   const void* dev_dout, uint64_t ld_dout, void* dev_dvalues, uint64_t ld_dvalues, float* dev_dweights,
                                   void* dev_workspace, uint64_t workspace_bytes, void* stream);

/* Dense product of n rows of `inputs` elements with a weight matrix, on the tensor cores (16-bit types, float32 sums). */
typedef struct pink_b200_product_config {
    uint32_t type;             /* PINK_B200_BF16 / F16: x, w, residual, out, z and their gradients                           */
    uint32_t inputs;           /* K                                                                                          */
    uint32_t outputs;          /* M                                                                                          */
    uint32_t by_input;         /* 0: w is [outputs][inputs]; 1: w is [inputs][outputs], as a table with a row per neuron is  */
    uint32_t activation;       /* PINK_B200_ACT_*                                                                            */
    uint32_t reserved;         /* 0                                                                                          */
    uint64_t n;                /* rows                                                                                       */
} pink_b200_product_config;

/* z = x W^T + bias (bias: [outputs] float32, nullable), out = act(z) + residual (nullable); sums, bias, activation and residual in
 * float32, out and z (nullable: kept for the backward pass) rounded once.  n, inputs and outputs below 2^31.
 * Scratch: the first call with size_only = 1 launches nothing and writes the bytes that exactly these arguments need to
 * *workspace_bytes; the call itself (size_only = 0) finds the size of dev_workspace there (16-byte aligned; NULL where 0 is enough).
 * Operands whose base is 16-byte aligned and whose leading dimension is a multiple of 16 are read in place (fastest: of 64);
 * others are copied into the workspace first where a tensor map cannot describe them or the copy pays.  Up to 8 rows need no
 * workspace.  dev_out may be dev_residual (same leading dimension). */
int pink_b200_op_product(const pink_b200_product_config* cfg, const void* dev_x, uint64_t ld_x, const void* dev_w, uint64_t ld_w,
                         const float* dev_bias, const void* dev_residual, uint64_t ld_residual, void* dev_out, uint64_t ld_out,
                         void* dev_z, uint64_t ld_z, void* dev_workspace, uint64_t* workspace_bytes, uint32_t size_only,
                         void* stream);

/* Its backward pass: dz = dout * act'(z) (z as kept by the forward call; not read without an activation), dx = dz W, dw = dz^T x in the
 * layout of w, dbias = column sums of dz in float32 ([outputs]); the residual's gradient is dout itself.  dx, dw, dbias may be
 * NULL.  dz enters the two products rounded to `type`, the column sums unrounded: half a step of dz, 2^-8 of it in bfloat16 and 2^-11
 * in float16.  In float16, behind an activation, a power of two common to the call keeps dz within the type's range: only what is 2^-28 of the
 * largest finite |dout| or less is rounded more coarsely.  Where z is an infinity, act' is its limit there (0 or 1).  Workspace as above. */
int pink_b200_op_product_backward(const pink_b200_product_config* cfg, const void* dev_dout, uint64_t ld_dout, const void* dev_x, uint64_t ld_x,
                                  const void* dev_w, uint64_t ld_w, const void* dev_z, uint64_t ld_z, void* dev_dx, uint64_t ld_dx,
                                  void* dev_dw, uint64_t ld_dw, float* dev_dbias, void* dev_workspace, uint64_t* workspace_bytes,
                                  uint32_t size_only, void* stream);

/* ---- training a head on a map -------------------------------------------------------
 * A head is a network whose inputs are images, their regions or a map's responses, and whose outputs are read beside the map's: it
 * learns values of the neurons, or the routes themselves, so that it answers without the rotations.  Beside the products above it takes
 * a norm of its inputs, gated hidden layers and a loss against the routes.  The rules above hold: the calls only launch kernels. */

/* Layer norm of n rows of `dims` elements (1 .. 2^24) of element type `type`: y = (x - mean) * rstd * weight + bias, with the row's mean
 * and rstd = 1 / sqrt(variance + eps), the variance over all `dims` elements (not dims - 1).  weight, bias: [dims] float32, nullable
 * (1 and 0).  dev_mean, dev_rstd: [n] float32, nullable, what the backward pass needs.  Sums are held in float32, those of squares about the
 * mean as rounded or a number within two standard deviations of it; y is rounded once.  A row with an infinity or a NaN becomes NaN; what a row
 * becomes whose sum or squares leave the range of float32 is not defined.  Rows on 16-byte boundaries are read, and written, fastest. */
int pink_b200_op_layer_norm(uint32_t type, uint32_t dims, uint64_t n, const void* dev_x, uint64_t ld_x, const float* dev_weight,
                            const float* dev_bias, float eps, void* dev_y, uint64_t ld_y, float* dev_mean, float* dev_rstd, void* stream);

/* Its backward pass, given x and the mean and rstd that the forward call wrote: with g = dy * weight and h = (x - mean) * rstd
 *   dx = rstd * (g - mean(g) - h * mean(g * h)) + residual   (residual, nullable: the gradient that arrives beside the norm, of `type`)
 *   dweight = column sums of dy * h, dbias = column sums of dy, float32, summed in a fixed order on a given device.
 * dx, or dweight and dbias together, may be NULL.  dev_dx may be dev_residual (same leading dimension).  dev_workspace: at least
 * pink_b200_layer_norm_workspace(...) bytes for the current device, 16-byte aligned; its content need not survive between calls. */
uint64_t pink_b200_layer_norm_workspace(uint32_t type, uint32_t dims, uint64_t n);
int pink_b200_op_layer_norm_backward(uint32_t type, uint32_t dims, uint64_t n, const void* dev_dy, uint64_t ld_dy, const void* dev_x,
                                     uint64_t ld_x, const float* dev_mean, const float* dev_rstd, const float* dev_weight,
                                     const void* dev_residual, uint64_t ld_residual, void* dev_dx, uint64_t ld_dx, float* dev_dweight,
                                     float* dev_dbias, void* dev_workspace, uint64_t workspace_bytes, void* stream);

/* Gated projections, the first half of a gated feed-forward block (the second is a product with the residual): g = x Wg^T + bg,
 * u = x Wu^T + bu, h = act(g) * u in one pass.  cfg as for pink_b200_op_product (inputs and outputs below 2^30); dev_gate and dev_up are Wg and Wu, both
 * [outputs][inputs], or with by_input = 1 both [inputs][outputs]; the biases are [outputs] float32, nullable.  Sums, biases, activation and
 * product in float32; h, and g and u (nullable each: kept for the backward pass) rounded once, h from the unrounded g and u.  Scratch as for pink_b200_op_product. */
int pink_b200_op_gated(const pink_b200_product_config* cfg, const void* dev_x, uint64_t ld_x, const void* dev_gate, uint64_t ld_gate,
                       const void* dev_up, uint64_t ld_up, const float* dev_gate_bias, const float* dev_up_bias, void* dev_h, uint64_t ld_h,
                       void* dev_g, uint64_t ld_g, void* dev_u, uint64_t ld_u, void* dev_workspace, uint64_t* workspace_bytes,
                       uint32_t size_only, void* stream);

/* Its backward pass, given g and u as the forward call kept them: dg = dh * u * act'(g), du = dh * act(g), dx = dg Wg + du Wu,
 * dgate = dg^T x and dup = du^T x in the layout of the weights, the bias gradients the column sums of dg and du in float32 ([outputs]).  dx, dgate with
 * dup, and the two bias gradients together may be NULL.  dg and du enter the products rounded to `type`, the column sums unrounded: half a step
 * of each, 2^-8 of it in bfloat16 and 2^-11 in float16.  In float16 a power of two common to the call keeps them within the type's range: only what is
 * 2^-28 of the largest finite one or less is rounded more coarsely.  Where g is an infinity, act and act' are their limits there; an infinite
 * g or u times a gradient that is zero is zero.  Workspace as above. */
int pink_b200_op_gated_backward(const pink_b200_product_config* cfg, const void* dev_dh, uint64_t ld_dh, const void* dev_x, uint64_t ld_x,
                                const void* dev_gate, uint64_t ld_gate, const void* dev_up, uint64_t ld_up, const void* dev_g, uint64_t ld_g,
                                const void* dev_u, uint64_t ld_u, void* dev_dx, uint64_t ld_dx, void* dev_dgate, uint64_t ld_dgate, void* dev_dup,
                                uint64_t ld_dup, float* dev_dgate_bias, float* dev_dup_bias, void* dev_workspace, uint64_t* workspace_bytes,
                                uint32_t size_only, void* stream);

/* What the targets of a distillation are. */
#define PINK_B200_TEACHER_WEIGHTS 0    /* probabilities, as the weights of a route        */
#define PINK_B200_TEACHER_LOGITS  1    /* logits, as a route's values times its slope     */

typedef struct pink_b200_distill_config {
    uint32_t n_neurons;        /* N: 1 .. 32768                                                                  */
    uint32_t top_k;            /* k: targets per image, 1 .. 32                                                  */
    uint32_t teacher;          /* PINK_B200_TEACHER_*                                                            */
    uint32_t rest;             /* 1 (weights only): what the weights leave of 1 belongs to the other neurons     */
    float temperature;         /* T: 0.001 .. 1000                                                               */
    float scale;               /* loss and gradient are multiplied by it; > 0.  T * T keeps gradients' size      */
} pink_b200_distill_config;

/* Distillation of a map's routes into n rows of scores ([n][ld_scores] of element type `type`), the divergence of the head's distribution
 * from the routes':
 *   takes part  a neuron whose mask (dev_mask: [N] bytes, nullable) is not zero and whose score is not -infinity.  A NaN, or a +infinity,
 *               of a neuron that is not masked makes its row's results NaN.
 *   q           softmax of score / T over the neurons that take part.
 *   targets     dev_neurons, dev_targets: [n][k], as pink_b200_op_route writes them.  A target is absent where its neuron is beyond N or
 *               takes no part, and where its weight is not above 0 (its logit not above -infinity); a logit of +infinity counts as the largest float.
 *   p           the weights; or the softmax of logit / T over the targets that are present.  A neuron listed twice counts twice: the gradient is that of its
 *               weights' sum, while the loss adds up p * log(p / q) of each entry, which is less than the sum's by the entropy of the split.
 *   loss        scale * (sum over the targets of p * log(p / q) + r * log(r / q_rest)); r = 0 without `rest`, otherwise 1 - sum of p, at
 *               least 0; q_rest is the sum of q over the neurons that take part and are not among the targets (without any: r = 0).
 * A row without targets has the loss 0 and the gradient 0, whatever its scores are.  dev_loss: [n] float32.
 * Without `rest`, weights that do not add up to 1 are taken as they are. */
int pink_b200_op_distill(const pink_b200_distill_config* cfg, uint64_t n, uint32_t type, const void* dev_scores, uint64_t ld_scores,
                         const uint8_t* dev_mask, const uint32_t* dev_neurons, const float* dev_targets, float* dev_loss, void* stream);

/* Its gradient with respect to the scores, given that of the losses (dev_dloss: [n], nullable: 1):
 *   dscores_e = dloss * scale / T * (q_e * (sum of p + r) - sum of p over the targets at e - r * q_e / q_rest where e is another)
 * [n][ld_dscores] of element type `type`, zero where a neuron takes no part.  dev_loss (nullable) receives the losses of the same pass: a
 * training step needs no forward call.  The targets have no gradient. */
int pink_b200_op_distill_backward(const pink_b200_distill_config* cfg, uint64_t n, uint32_t type, const void* dev_scores, uint64_t ld_scores,
                                  const uint8_t* dev_mask, const uint32_t* dev_neurons, const float* dev_targets, const float* dev_dloss,
                                  void* dev_dscores, uint64_t ld_dscores, float* dev_loss, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* PINK_B200_H */
