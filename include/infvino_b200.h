/*
 * infvino_b200 - C ABI of the B200 plan executor (drop-in for infvino's
 * OpenCL `PlanModel` / `ClBackend`).
 *
 * Plain C types only: handles are opaque pointers, tensors are raw pointers plus
 * element counts, CUDA streams are passed as `void *` (a cudaStream_t).  Every
 * call returns an ivc_status; the message of the last failure on a handle is
 * available from ivc_last_error().  Calls on one handle are serialised
 * internally (as `ClBackend::infer` is, src/ClBackend.cpp:33 in the reference).
 *
 * Batching: plans declare batch 1 (dim 0 of every activation).  A handle is
 * created for `max_batch` images; each call names the batch it processes and
 * every buffer holds `batch * numel` elements, image-major.
 *
 * Reference interfaces each entry point replaces (paths inside the reference):
 *   ivc_create ............ PlanModel::PlanModel  include/infvino/PlanModel.hpp:57-59
 *                            ClBackend::ClBackend  include/infvino/ClBackend.hpp:32
 *   ivc_input_* / output_*  PlanModel::inputName/inputDims/inputNumel/outputCount/
 *                            outputName/outputDims/outputNumel  PlanModel.hpp:64-73
 *   ivc_tensor_numel ....... PlanModel::tensorNumel  PlanModel.hpp:85-86
 *   ivc_infer_f32 .......... ClBackend::infer(const float*, size_t)  ClBackend.hpp:38-39
 *   ivc_set_input_f16 ...... PlanModel::setInput(const void*)  PlanModel.hpp:75-76
 *   ivc_run ................ PlanModel::run()  PlanModel.hpp:77-78
 *   ivc_run_async .......... PlanModel::run() without the final finish (PlanModel.cpp:4175)
 *   ivc_read_output_f16 .... PlanModel::readOutput(size_t, void*)  PlanModel.hpp:79-80
 *   ivc_read_tensor_f16 .... PlanModel::readTensor(name, void*)  PlanModel.hpp:82-84
 *   ivc_last_infer_ms ...... ClBackend::lastInferMs / PlanModel::lastRunMs
 *                            ClBackend.hpp:41, PlanModel.hpp:190-191
 *   ivc_profile / ivc_step_* PlanModel::profile() / PlanProfile  PlanModel.hpp:204-224
 *   ivc_pool_stats ......... PlanModel::poolRequestedBytes/poolAllocatedBytes/
 *                            poolBufferCount  PlanModel.hpp:94-97
 *   ivc_infer_f16_device ... (new) zero-copy device-pointer inference on a caller stream
 *   ivc_set_input_bgr_u8 / ivc_infer_bgr_u8
 *                            Preprocessor::operator() src/Preprocess.cpp:13-77 (+ ClBackend::infer), on the device
 *   ivc_decode_pose ........ PoseDecoder::decode + nmsPerClass + nms, on the device
 *                            src/Decoders.cpp:33-65,127-179, src/Nms.cpp:10-55
 *   ivc_destroy ............ PlanModel::~PlanModel / ClBackend destructor
 */
#ifndef INFVINO_B200_H_
#define INFVINO_B200_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ivc_model ivc_model;

typedef enum ivc_status {
  IVC_OK = 0,
  IVC_ERR_ARGUMENT = 1,   /* bad pointer / index / batch */
  IVC_ERR_PLAN = 2,       /* plan parse, missing init, unknown op (reference: std::runtime_error) */
  IVC_ERR_CUDA = 3,       /* CUDA runtime / device failure */
  IVC_ERR_NUMEL = 4,      /* input element count does not match the plan */
  IVC_ERR_KERNEL = 5,     /* a kernel reported a bounded-wait timeout (status word) */
  IVC_ERR_NOT_FOUND = 6   /* unknown tensor name */
} ivc_status;

/* creation flags */
#define IVC_FLAG_NO_GRAPH 0x1u        /* eager launches instead of CUDA graph replay */
#define IVC_FLAG_NO_FUSION 0x2u       /* skip concat->conv1x1 / residual load-time rewrites */
#define IVC_FLAG_DRY_RUN 0x4u         /* host only: parse, layout, allocate; no GPU is touched */
#define IVC_FLAG_NO_TENSOR_CORES 0x8u /* convolutions on the CUDA-core direct kernel (diagnostic) */
#define IVC_FLAG_NO_POOL 0x10u        /* no activation memory reuse, every tensor stays readable
                                         (reference INFVINO_NO_POOL, src/PlanModel.cpp:887) */
#define IVC_FLAG_NO_HALO 0x20u        /* diagnostic: 3x3 stride-1 convolutions load one box per tap
                                         instead of one halo box per channel chunk */
#define IVC_FLAG_NO_PDL 0x40u         /* diagnostic: kernels launched without programmatic dependent
                                         launch (each waits for the previous grid to finish) */
#define IVC_FLAG_NO_JIT 0x80u         /* diagnostic: the fused decode tail runs on the interpreting
                                         kernel instead of its load-time compiled (NVRTC) form */
#define IVC_FLAG_NO_TUNE 0x100u       /* convolution tile geometry from the cost model alone (no timing
                                         of candidate geometries at the first run of a batch size) */
#define IVC_FLAG_SERIAL 0x200u        /* every step on one stream: the captured graph has no concurrent
                                         branches (and activations may share more memory) */

/* Loads `plan_path` (+ its init_*.bin files) onto CUDA device `device_ordinal`. */
int ivc_create(const char *plan_path, int device_ordinal, int max_batch, unsigned flags, ivc_model **out);
void ivc_destroy(ivc_model *m);
/* Message of the last failed call on `m`; with m == NULL, of the last failed ivc_create. */
const char *ivc_last_error(const ivc_model *m);

int ivc_input_name(const ivc_model *m, const char **name);
int ivc_input_dims(const ivc_model *m, int64_t *dims, int max_rank, int *rank);
int64_t ivc_input_numel(const ivc_model *m);
int ivc_output_count(const ivc_model *m);
int ivc_output_name(const ivc_model *m, int i, const char **name);
int ivc_output_dims(const ivc_model *m, int i, int64_t *dims, int max_rank, int *rank);
int64_t ivc_output_numel(const ivc_model *m, int i);
/* per-image element count of any declared tensor, 0 if unknown */
int64_t ivc_tensor_numel(const ivc_model *m, const char *name);
int ivc_max_batch(const ivc_model *m);

/* ClBackend::infer: `input` holds batch*input_numel f32 values (host memory,
 * pinned or pageable); converted to fp16 with the reference's truncating cast,
 * run, and every output written as f32 to outputs[i] (batch*output_numel(i)
 * values, host memory).  Synchronous.  Batches of 32 or more are pipelined in
 * chunks, and half of their images are cast on the host by a process-wide
 * pool of worker threads (one per CPU of the process's affinity mask, up to
 * 16, created at the first such call), so that fewer bytes cross PCIe; the
 * first call also pins two chunk buffers. */
int ivc_infer_f32(ivc_model *m, const float *input, size_t numel, int batch, float *const *outputs);

/* PlanModel-style split calls (fp16 host buffers, synchronous). */
int ivc_set_input_f16(ivc_model *m, const uint16_t *input_f16, int batch);
int ivc_run(ivc_model *m, int batch);
/* PlanModel::run without the host wait: enqueues the network for the input set
 * last, on `stream` (NULL = the handle's stream). */
int ivc_run_async(ivc_model *m, int batch, void *stream);
int ivc_read_output_f16(ivc_model *m, int i, uint16_t *dst, int batch);
/* Copies tensor `name` for `batch` images in plan (NCHW) order; IVC_ERR_NOT_FOUND if unknown. */
int ivc_read_tensor_f16(ivc_model *m, const char *name, uint16_t *dst, int batch);

/* Image preprocessing on the device (replaces the host-side
 * Preprocessor::operator(), src/Preprocess.cpp:13-77, and the truncating cast
 * of ClBackend::infer).  Settings as infvino::PreprocessConfig
 * (include/infvino/Preprocess.hpp:40-48); the input size is the plan's input. */
typedef struct ivc_preprocess {
  int letterbox;        /* 1: keep the aspect ratio and pad with 114 (the default); 0: plain resize */
  int to_rgb;           /* 1: BGR -> RGB (the default) */
  int normalize;        /* 1: x 1/255 (the default) */
  int n_mean, n_std;    /* entries of mean / std in use (0: none), applied after /255 */
  float mean[3], std[3];
} ivc_preprocess;

/* `batch` 8-bit BGR frames (height x width x 3, rows `row_stride` bytes apart,
 * frames height * row_stride bytes apart) in host memory (pinned or pageable),
 * or in device memory when frames_on_device is nonzero, become the network
 * input: letterbox + cv::resize INTER_LINEAR (OpenCV's 8-bit arithmetic,
 * bit-exact) + 114 border + blobFromImage + mean / std + the reference's
 * truncating f32 -> f16 cast, in one kernel.  cfg NULL: the defaults above.
 * letterbox (host, [batch][scale, pad_left, pad_top]) or NULL receives what
 * Preprocessor reports in LetterboxInfo.  Synchronous. */
int ivc_set_input_bgr_u8(ivc_model *m, const uint8_t *frames, int batch, int height, int width, size_t row_stride,
                         int frames_on_device, const ivc_preprocess *cfg, float *letterbox);
/* End to end from 8-bit BGR frames in host memory to f32 outputs in host
 * memory (Preprocessor + ClBackend::infer in one call): large batches are
 * pipelined in chunks (frames copied in, preprocessed, run, results copied
 * out, overlapped).  Synchronous. */
int ivc_infer_bgr_u8(ivc_model *m, const uint8_t *frames, int batch, int height, int width, size_t row_stride,
                     const ivc_preprocess *cfg, float *const *outputs, float *letterbox);

/* Pose decode + greedy NMS of output 0 of the last run, on the device, for
 * `batch` images (replaces the host-side PoseDecoder::decode with
 * nmsPerClass, src/Decoders.cpp:127-179 and :33-65, and nms / iou,
 * src/Nms.cpp:10-55).  Candidates are anchors whose score is not below
 * `conf`; boxes and keypoints are mapped through the letterbox
 * (include/infvino/Preprocess.hpp:24-35; `letterbox` is [batch][scale,
 * pad_left, pad_top] in host memory, or NULL for scale 1 and no padding);
 * greedy suppression at IoU above `iou` in descending score (ties by anchor
 * index, the reference's stable sort); the keep list is then re-sorted by
 * score with std::sort and cut at `max_det`, as the reference does, so equal
 * scores come out in the order that (unstable) sort leaves them.  Results in
 * host memory:
 * counts[b] detections for image b, detection k at
 * dets[(b * max_det + k) * (6 + 2 * nk)]: anchor index, score, x, y, w, h,
 * then x, y of each keypoint.  nk <= 0 infers the keypoint count from the
 * output's channels as (C - 5) / kdims (kdims <= 0: 3).  The output must be
 * channel-major [1, 5 + nk * kdims, A] with A <= 16384.  Synchronous. */
int ivc_decode_pose(ivc_model *m, int batch, float conf, float iou, int max_det, int nk, int kdims,
                    const float *letterbox, int *counts, float *dets);
/* ivc_read_tensor_f16 without any allocation (no counterpart in the reference).
 * The NHWC -> NCHW relayout is staged through a static 4 MiB device buffer per
 * device instead of a scratch buffer grown with cudaMalloc; a tensor that needs
 * more than 4 MiB for `batch` images fails with IVC_ERR_ARGUMENT.  For callers
 * that must not allocate or free device memory after set-up: a process whose
 * device memory is owned by another allocator, or a diagnostic read inside a
 * latency-critical loop (cudaFree synchronises the whole device).  Make the
 * first call on each device before any stream capture (it resolves the
 * buffer's address, which may load the module).  Overlapping calls on one
 * device (from any handle) share the buffer and race. */
int ivc_read_tensor_f16_noalloc(ivc_model *m, const char *name, uint16_t *dst, int batch);

/* Zero-copy: device fp16 input / outputs, enqueued on `stream` (cudaStream_t,
 * NULL = the handle's stream) without host synchronisation. */
int ivc_infer_f16_device(ivc_model *m, const void *d_input, int batch, void *const *d_outputs, void *stream);
/* Device f32 input (truncating cast on the device) -> device f32 outputs, asynchronous. */
int ivc_infer_f32_device(ivc_model *m, const float *d_input, int batch, float *const *d_outputs, void *stream);
/* Binds the handle to a caller stream (NULL restores a private stream). */
int ivc_set_stream(ivc_model *m, void *stream);
int ivc_synchronize(ivc_model *m);
double ivc_last_infer_ms(const ivc_model *m);

/* Profiling: eager run with CUDA events around every kernel launch. */
int ivc_step_count(const ivc_model *m);
int ivc_step_info(const ivc_model *m, int i, const char **name, const char **family, double *flops_per_image,
                  double *act_bytes_per_image, double *fixed_bytes);
int ivc_profile(ivc_model *m, int batch, float *step_ms, int n);
/* Number of kernel launches one ivc_run(batch) performs (kernel nodes of its CUDA graph). */
int ivc_launch_count(ivc_model *m, int batch, int *count);

/* Diagnostic (no counterpart in the reference): settings of the convolution
 * kernels' bounded waits.  `limit_cycles` is the limit of every working wait
 * in SM clocks (the default is about 2 s); with `probe` nonzero each conv CTA
 * first waits on a barrier that nothing arrives on, so that wait runs out, the
 * kernel drains its copies and MMAs, releases TMEM and reports its status, and
 * the next synchronising call returns IVC_ERR_KERNEL.  Lets a test exercise the
 * timeout path without any GPU fault; the handle stays usable.  Takes effect
 * from the next run (captured graphs are captured again). */
int ivc_debug_conv_wait(ivc_model *m, long long limit_cycles, int probe);

/* Activation pool statistics (bytes at max_batch). */
int ivc_pool_stats(const ivc_model *m, int64_t *requested_bytes, int64_t *arena_bytes, int64_t *weight_bytes,
                   int *roots, int *views, int *nhwc_tensors, int *fusions_concat, int *fusions_res);
/* Human-readable dump of tensors (layout, arena offset, lifetime) and launches. */
int ivc_describe(const ivc_model *m, char *buf, size_t cap);

/* Properties of CUDA device `device_ordinal`, for the reference's DeviceInfo
 * (include/infvino/Device.hpp:16-26, describeDevice): name, multiprocessor
 * count (DeviceInfo::eu), clock (DeviceInfo::clock_mhz), compute capability,
 * memory, and the number of devices (DeviceInfo::available). */
typedef struct ivc_device_props {
  char name[256];
  int multiprocessors;
  int clock_mhz;
  int cc_major, cc_minor;
  int64_t total_mem_bytes;
  int device_count;
  int runtime_version;  /* CUDA runtime, e.g. 12090 */
} ivc_device_props;
int ivc_device_properties(int device_ordinal, ivc_device_props *out);

/* Host conversions with the reference's semantics (include/infvino/Half.hpp:14-49). */
void ivc_f32_to_f16(const float *in, uint16_t *out, size_t n);
void ivc_f16_to_f32(const uint16_t *in, float *out, size_t n);

/* ------------------------------------------------------------------------
 * Language-model operators: rotary positions, a paged key/value cache held in
 * 8 bits, the attention over it, products in microscaled 4-bit numbers and the
 * choice of tokens, for a decoder that follows a network of this library (its
 * outputs become tokens).  Inference only.
 *
 * All tensors are device memory of the handle's device; nothing is copied and
 * no call waits for the device.  `stream` is a cudaStream_t; NULL is the
 * legacy default stream.  Argument errors that the host can see come back as
 * IVC_ERR_ARGUMENT.  What only the device sees is skipped by the kernels, which
 * set the handle's status word: ivc_kv_synchronize then returns IVC_ERR_KERNEL
 * and clears it.  Skipped is: of a token with a position outside the rotary
 * table everything (no row, code or scale of it is written); of a token without
 * a place in the cache (a page number outside it, offsets or lengths that do
 * not fit) the codes, or the row that would be read; of attention, a sequence
 * whose offsets or length do not fit, and the keys in a page outside the cache,
 * as if they were hidden.  The others of the call are as they would be alone.
 *
 * Calls may be captured into a CUDA graph, ivc_kv_attend and
 * ivc_kv_attend_shared once the stream has had one call of either or of
 * ivc_kv_reserve (each stream has its own workspace, so calls on several streams
 * may run at the same time; cudaStreamPerThread is another stream in every
 * thread).  A graph with one of these uses the workspace of the stream that it
 * was captured on: its replays must not overlap one another, other graphs' from
 * that stream, or eager calls on it. */
typedef struct ivc_kv ivc_kv;

typedef enum ivc_dtype { IVC_F16 = 0, IVC_BF16 = 1, IVC_F32 = 2 /* logits only */ } ivc_dtype;

/* [tokens][heads][head_dim] of the call's dtype; strides in elements, the last
 * dimension dense.  Any 2-byte alignment works; 16-byte alignment of data and
 * strides takes the vector path.  Rows that are written do not overlap. */
typedef struct ivc_rows {
  void *data;
  int64_t token_stride, head_stride;
} ivc_rows;

/* One layer's cache, in the caller's memory.  Codes [pages][kv_heads]
 * [page_size][head_dim] in -127..127; a value is code * scale, one scale (a
 * power of two, as ivc_kv_append writes it; never negative, infinite or NaN where
 * it is read) for each IVC_KV_BLOCK tokens of a page and head:
 * [pages][kv_heads][page_size / IVC_KV_BLOCK].  page_size is a
 * multiple of IVC_KV_BLOCK, head_dim 64 or 128, k and v 16-byte aligned. */
#define IVC_KV_BLOCK 16
typedef struct ivc_kv_cache {
  int8_t *k, *v;
  float *k_scale, *v_scale;
  int64_t pages;
  int page_size, kv_heads, head_dim;
} ivc_kv_cache;

/* The sequences of a call.  Sequence b owns the packed tokens offsets[b] ..
 * offsets[b + 1] - 1 (offsets [batch + 1], from 0, not falling; none or more
 * each).  at[b]: append and read: the cache position of the first of them;
 * attend: how many tokens the cache holds, the call's own included (they are
 * the last ones).  The token at position p is in page
 * pages[b * pages_per_seq + p / page_size].  Device memory, int32. */
typedef struct ivc_kv_seqs {
  int batch;
  int64_t tokens;
  const int32_t *offsets, *at, *pages;
  int pages_per_seq;
} ivc_kv_seqs;

/* Rotary positions with `axes` (1..4) position numbers for each token, e.g.
 * time, height, width: pos[a * pos_stride + token].  Pair i of a head, of
 * `pairs` (2 * pairs <= head_dim; the rest of the head is left as it is), is
 * elements (i, i + pairs), or (2i, 2i + 1) if interleaved.  It turns by the
 * angle whose cosine and sine are table[position on axis axis_of[i]][i]:
 * table [positions][pairs][2], device memory.  axis_of: host memory [pairs],
 * or NULL for axis 0 throughout. */
#define IVC_KV_MAX_PAIRS 128
typedef struct ivc_rotary {
  const float *table;
  int64_t positions;
  int pairs, axes, interleaved;
  const int32_t *pos;
  int64_t pos_stride;
  const uint8_t *axis_of;
} ivc_rotary;

int ivc_kv_create(int device_ordinal, ivc_kv **out);
void ivc_kv_destroy(ivc_kv *h);
/* Message of the calling thread's last failed call on `h` (for a thread without
 * one, of any thread's); with h == NULL, of its last failed ivc_kv_create.  Valid
 * until the thread's next call of this function. */
const char *ivc_kv_last_error(const ivc_kv *h);
/* Waits for `stream` and reports what the kernels found wrong, once.  There is
 * one status word for a handle: with several streams the first call to come
 * reports the first error of any of them, and clears the word (use a handle for
 * each stream where that matters).  Other threads' calls do not wait for it. */
int ivc_kv_synchronize(ivc_kv *h, void *stream);
/* Allocates the stream's attention workspace (else its first ivc_kv_attend does). */
int ivc_kv_reserve(ivc_kv *h, void *stream);
/* Waits for the stream and frees its attention workspace (some 40 MB; else the
 * handle keeps it to its end).  To be called before a stream is destroyed.
 * Graphs captured on the stream must not be replayed after it. */
int ivc_kv_release(ivc_kv *h, void *stream);

/* Diagnostic: with limit_cycles above 0 every other CTA of ivc_kv_attend's
 * kernel for many queries first waits so many SM clocks (2 M are about 1 ms)
 * for what never comes, and gives up as after any wait that runs out: the
 * call's results are not valid, and ivc_kv_synchronize returns IVC_ERR_KERNEL.
 * Calls after that (0 again) are as if it had not been. */
int ivc_debug_kv_probe(ivc_kv *h, long long limit_cycles);

/* Fills a rotary table: the angle of position p and pair i is p * inv_freq[i]
 * (host memory [pairs]), computed in 64 bits and rounded once. */
int ivc_kv_rope_table(ivc_kv *h, const double *inv_freq, int pairs, int64_t positions, float *table, void *stream);
/* out = x with its pairs turned, in f32, rounded once; out may be x. */
int ivc_kv_rope(ivc_kv *h, int dtype, int64_t tokens, int heads, int head_dim, const ivc_rows *x, const ivc_rows *out,
                const ivc_rotary *rotary, void *stream);
/* Appends keys (turned by `rotary`, unless NULL) and values to the cache, and
 * turns q into q_out (q_heads 0: no queries) in the same launch.
 * A block's exponent is the least e with |x| <= 127 * 2^e (in -120..121) over
 * its new tokens; if the block already holds tokens of the sequence, their
 * exponent if that is larger, and when e grows their codes c become
 * round(c * 2^(old - e)), ties to even, as the new codes are round(x * 2^-e).
 * So growth costs at most one rounding each time and the errors of all add up
 * to less than one final step.  NaN is held as 0, an infinity as the largest
 * code of its sign; neither takes part in e. */
int ivc_kv_append(ivc_kv *h, const ivc_kv_cache *cache, const ivc_kv_seqs *seqs, int dtype, const ivc_rows *k,
                  const ivc_rows *v, const ivc_rotary *rotary, int q_heads, const ivc_rows *q, const ivc_rows *q_out,
                  void *stream);
/* The cache's values of the sequences' tokens into k and v (either may be NULL). */
int ivc_kv_read(ivc_kv *h, const ivc_kv_cache *cache, const ivc_kv_seqs *seqs, int dtype, const ivc_rows *k,
                const ivc_rows *v, void *stream);
/* out = softmax(scale * q k^T) v over the cache.  The query at position p sees
 * the keys j <= p, with window > 0 only those with p - j < window or
 * j < sinks.  q_heads is a multiple of kv_heads; query head h reads kv head
 * h / (q_heads / kv_heads).  A row that sees nothing gives 0.  max_new: at
 * least the largest number of new tokens of one sequence.  Scores, maxima and
 * sums are in f32; a weight meets the values as a half, with 11 bits down to
 * 2^-22 of a row's largest weight times value scale and fewer below. */
int ivc_kv_attend(ivc_kv *h, const ivc_kv_cache *cache, const ivc_kv_seqs *seqs, int dtype, int q_heads, int max_new,
                  const ivc_rows *q, const ivc_rows *out, float scale, int window, int sinks, void *stream);

/* Sequences that begin alike: group g is the sequences first[g] ..
 * first[g + 1] - 1 of a call (first [count + 1], from 0 to batch, rising), and
 * their first shared[g] tokens (whole pages; 0: none) are in the pages that the
 * group's first sequence has for them.  Device memory, int32. */
typedef struct ivc_kv_groups {
  int count;
  const int32_t *first, *shared;
} ivc_kv_groups;
/* ivc_kv_attend without a window, for groups of sequences with a common
 * beginning (samples or questions over the same frames): its keys and values are
 * read once for all of a group's queries, with ivc_kv_attend's roundings.  Every sequence's new tokens come
 * after it (lens[b] - new tokens >= shared[g]); a sequence's own pages for the
 * first shared[g] tokens are not looked at.  A group whose sequences, or whose
 * shared[g], do not fit is skipped, as is a sequence that ends inside the
 * beginning.  scratch: at least tokens * q_heads * (head_dim + 2) floats, 16-byte
 * aligned, of nobody else until the call has run (memory of q, out or the cache's
 * codes and scales is refused). */
int ivc_kv_attend_shared(ivc_kv *h, const ivc_kv_cache *cache, const ivc_kv_seqs *seqs, const ivc_kv_groups *groups,
                         int dtype, int q_heads, int max_new, const ivc_rows *q, const ivc_rows *out, float scale,
                         float *scratch, int64_t scratch_floats, void *stream);

/* The next token of each row of logits [rows][vocab] (IVC_F16, IVC_BF16 or
 * IVC_F32, rows row_stride elements apart, vocab at most 500000). */
typedef struct ivc_logits {
  const void *data;
  int dtype;
  int64_t rows, vocab, row_stride;
} ivc_logits;
/* For each row, device memory: a random number u in [0, 1), a temperature, and the
 * filters; those that are NULL are off (temperature: 1). */
typedef struct ivc_sampling {
  const float *u, *temperature;
  const int32_t *top_k;
  const float *top_p, *min_p;
} ivc_sampling;
/* Token i has the weight w_i = e^((x_i - x_max) / temperature), and the tokens are
 * ordered by their logits, equal ones by their numbers.  Kept are, one filter after
 * the other, the first top_k (0 and below: all); of them the shortest beginning
 * with at least top_p of their weight (1 and above, NaN: all); of them those with
 * w_i >= min_p (0 and below, NaN: all); always the first.  tokens[row] is the least
 * i for which the weights of the kept tokens up to i exceed u times the weight of
 * all kept ones, probs[row] (NULL: not wanted) its share of that.  With a
 * temperature that is not above 0 it is the first in order, with probability 1.
 * A logit of NaN counts as -inf; where one is +inf, only those have a weight; a
 * row of -inf alone gives token -1 with probability 0.  Weights and sums are in 64
 * bits; weights below 2^-60 count as 0.  u is taken into [0, 1) (NaN: 0).  The order
 * of the sums goes by vocab, the number of rows, the device and the row's address
 * modulo 16: with these the same, so is every bit; otherwise a row within a rounding
 * of a border may get a neighbouring cut or token. */
int ivc_kv_sample(ivc_kv *h, const ivc_logits *logits, const ivc_sampling *how, int32_t *tokens, float *probs,
                  void *stream);

/* A matrix [rows][width] of microscaled 4-bit numbers (the OCP format MXFP4),
 * width a multiple of 32.  codes [rows][width / 2], the lower four bits first:
 * sign, two bits of exponent, one of mantissa (0, 0.5, 1, 1.5, 2, 3, 4, 6).
 * Scales are powers of two, 2^(e - 127), for each IVC_MX4_BLOCK values of a row
 * (e = 255: NaN), laid out as the tensor cores read them: the byte e of block b
 * of row r is scales[r / 128][b / 4][r % 32][r % 128 / 32][b % 4], of
 * [ceil(rows / 128)][ceil(width / 128)][32][4][4]; bytes without a row or block
 * are 0.  Device memory; both 16-byte aligned. */
#define IVC_MX4_BLOCK 32
typedef struct ivc_mx4 {
  uint8_t *codes, *scales;
  int64_t rows, width;
} ivc_mx4;
/* m = x [rows][width] (IVC_F16 or IVC_BF16, rows x_stride elements apart), its
 * first `rows` rows: e - 127 is the exponent of a block's largest magnitude less 2
 * (at least -127), and codes are x 2^(127 - e), rounded to the nearest, ties to
 * even, at most 6.  NaN is held as 0, an infinity as the largest code of its sign;
 * neither takes part in e.  The matrix's rows behind these stay as they are.  m
 * shares no memory with x. */
int ivc_kv_mx4_quantize(ivc_kv *h, int dtype, const void *x, int64_t rows, int64_t x_stride, const ivc_mx4 *m,
                        void *stream);
/* out = the values of m's first `rows` rows, rounded once (out_stride elements
 * apart; it shares no memory with m). */
int ivc_kv_mx4_read(ivc_kv *h, const ivc_mx4 *m, int64_t rows, int dtype, void *out, int64_t out_stride, void *stream);
/* out [rows][w->rows] = X W^T, summed in f32 and rounded once: W is w; X is the
 * first `rows` rows of xq if x is NULL, else x [rows][width] (x_dtype), quantised as
 * ivc_kv_mx4_quantize does it: xq is room for that then, of nobody else until
 * the call has run, and what it holds afterwards is not defined.  out, and the room
 * for x, share no memory with the others (rows may lie between one another's).
 * Outputs of out_dtype (IVC_F16 or IVC_BF16). */
int ivc_kv_mx4_linear(ivc_kv *h, int x_dtype, const void *x, int64_t rows, int64_t x_stride, const ivc_mx4 *xq,
                      const ivc_mx4 *w, int out_dtype, void *out, int64_t out_stride, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* INFVINO_B200_H_ */
