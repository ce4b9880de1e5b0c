/*
 * mpserve_amd — MI355X (gfx950) FP8 + Huffman-sidecar weight path and MXFP4 operators, C ABI.
 *
 * Plain pointers and sizes only. Every pointer named "device" is HIP device
 * memory on the current device; host pointers are named so. All entry points
 * return MPS_OK (0) or a negative MPS_ERR_* code; mps_last_error() gives the
 * message of the last failure on the calling thread.
 *
 * Sidecar format: the one MPServe's builder writes
 * (reference kernel/build_huffman.cu:292-969, scripts/compress_llm_fp8_huffman.py:284-306).
 */
#ifndef MPSERVE_AMD_H
#define MPSERVE_AMD_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MPS_OK 0
#define MPS_ERR_INVALID_ARGUMENT (-1) /* maps to Python ValueError (std::invalid_argument in the reference) */
#define MPS_ERR_RUNTIME (-2)          /* maps to Python RuntimeError */
#define MPS_ERR_HIP (-3)              /* a HIP runtime call failed */
#define MPS_ERR_NO_MEMORY (-4)

/* Device-side integrity flags a decode records (see mps_fp8_read_status). */
#define MPS_STATUS_BAD_BUCKET 0x1u   /* row range / column range outside the tensor */
#define MPS_STATUS_BAD_ROW 0x2u      /* a row index outside [0, n) */
#define MPS_STATUS_BAD_TABLE 0x4u    /* a bucket_table gid outside [-1, G) */
#define MPS_STATUS_DESYNC 0x8u       /* a lane ended at a bit other than the next lane's start */

/* One FP8 tensor and its sidecar, all device pointers, as stored by the
 * reference's compress script (huff_* tensors) with the decode call's dtype
 * views (reference scripts/mpserve_vllm_fp8_huffman.py:457-472). */
typedef struct mps_fp8_tensor {
  const uint8_t *fp8;                    /* [n*m]            huff_fp8_u8 */
  const uint64_t *bitstream;             /* [bitstream_words] huff_bitstream_u64 */
  int64_t bitstream_words;
  const uint16_t *decode_syms;           /* [num_tables,128] huff_decode_syms_u16 */
  const uint8_t *decode_lens;            /* [num_tables,64]  huff_decode_lens_u8 (packed 4-bit) */
  int64_t num_tables;
  const int32_t *bucket_table;           /* [num_buckets,256] fp8 byte -> table id or -1 */
  const int32_t *bucket_col_start;       /* [num_buckets] */
  const int32_t *bucket_col_len;         /* [num_buckets] */
  const int32_t *bucket_row_offsets;     /* [num_buckets+1] into row_indices */
  const int32_t *row_indices;            /* [num_row_indices] */
  int64_t num_row_indices;
  const uint32_t *bucket_thread_startbit;/* [num_buckets, k+1] lane start bits, relative */
  const int64_t *bucket_bit_base;        /* [num_buckets+1] bucket base bits (64-aligned) */
  int64_t num_buckets;
  int64_t k;                             /* substreams (lanes) per bucket, 1..1024 */
  int64_t n, m;                          /* output shape [n, m] */
  uint16_t *out;                         /* [n*m] BF16 bit patterns (device) */
} mps_fp8_tensor;

/* Message of the last failed call on this thread ("" if none). */
const char *mps_last_error(void);

/* HIP clock rate (kHz) of `device`.
 * Replaces MPServe_cuda.cuda_clock_rate_khz (reference kernel/wrapper.cpp:133-141). */
int mps_clock_rate_khz(int device, int64_t *khz_out);

/* Decode one tensor: out[n,m] = BF16 rebuilt from FP8 bytes + sidecar, on `stream`
 * (a hipStream_t; NULL = the legacy default stream). Lossless: reads the raw
 * 16 bits after ESC codes, and walks columns as e % col_len.
 * Replaces huffman_cpp::huffman_decode_fp8_entry (reference kernel/decode_huffman.cu:591-758,
 * bound as MPServe_cuda.huffman_decode_fp8 at kernel/wrapper.cpp:456-503); the
 * shape/dtype checks of that entry are done by the caller, which knows dtypes.
 * max_len must be 7. Asynchronous: returns after the launch. */
int mps_fp8_decode(const mps_fp8_tensor *tensor, int64_t max_len, void *stream);

/* Batched decode plan: one launch decodes many tensors (a layer, a model).
 * Creation first synchronises `stream` (the caller's stream, which may still
 * be writing the sidecars), then reads each tensor's bucket row offsets,
 * column ranges and bit bases to order the work largest first and to build
 * one work record per bucket, and copies the descriptors into one device
 * allocation the plan owns (with its own status word). When the buckets are
 * few or uneven for the device's CUs, large buckets are split into ranges of
 * rows (of steps of k elements, where the columns are no multiple of k): a
 * kernel on `stream` walks their substreams' code lengths once and records
 * each substream's bit position at every range's start (the lane checkpoints,
 * also owned by the plan). Small buckets whose table ids are equal (128 x 128
 * blocks of one scale) are grouped into items that set the tables up once. A
 * sidecar whose bucket metadata, row indices, start bits, tables, FP8 bytes or
 * bitstream is rewritten needs a new plan in either case. The pointed-to sidecars must stay alive while the
 * plan is used. Launches are persistent: one workgroup per CU takes work
 * items from a queue in the plan's memory, which each launch leaves as it
 * found it. The plan holds 32 such queues and gives each stream that launches
 * it (mps_fp8_plan_decode and mps_fp8_plan_decode_into alike) its own at the
 * stream's first launch, so launches on different streams may overlap, and a
 * launch captured into a graph replays with the queue of the stream it was
 * captured on (a replay must then not overlap an eager launch on that same
 * stream). A 33rd stream is refused with MPS_ERR_RUNTIME. Decodes are
 * asynchronous on their stream and OR their MPS_STATUS_* flags into the
 * plan's status word (mps_fp8_plan_read_status).
 * No counterpart in the reference, which launches once per tensor
 * (kernel/decode_huffman.cu:739); it serves its apply() and model loading paths
 * (scripts/mpserve_vllm_fp8_huffman.py:491-557). */
typedef struct mps_fp8_plan mps_fp8_plan;
int mps_fp8_plan_create(const mps_fp8_tensor *tensors, int64_t count, void *stream, mps_fp8_plan **plan_out);
int mps_fp8_plan_decode(mps_fp8_plan *plan, void *stream);
/* Decode the plan into a buffer laid out like the outputs it was created
 * with, moved to `out`: every tensor's output moves by (out - the first
 * tensor's output at creation), in BF16 elements. A plan of one tensor decodes
 * into any n*m buffer; a plan whose tensors' outputs are row slices of one
 * weight decodes into any buffer of that weight's size. The flags go to the
 * device status word (mps_fp8_read_status), as a single-tensor decode's do.
 * This serves the drop-in decode op's per-sidecar plan cache and the vLLM
 * method's scratch slots. */
int mps_fp8_plan_decode_into(mps_fp8_plan *plan, uint16_t *out, void *stream);
/* The plan's work list (for profiling tools): work items (buckets, runs of
 * them, and the ranges of the buckets it split), bytes of LDS per workgroup. */
int mps_fp8_plan_info(const mps_fp8_plan *plan, int64_t *work_items, int64_t *lds_bytes);
/* Read and clear the plan's MPS_STATUS_* flags; synchronises `stream` first. */
int mps_fp8_plan_read_status(mps_fp8_plan *plan, void *stream, uint32_t *status_out);
int mps_fp8_plan_destroy(mps_fp8_plan *plan);

/* Allocation-free batched decode: decodes `count` tensors (at most 1024, with
 * at most 63,100 buckets in all) in one persistent launch, as a plan would,
 * but without creating one. It calls no hipMalloc, hipFree or other
 * allocating routine and does not synchronise: the descriptors (copied from
 * the host array on `stream`) and one work record per bucket go into a static
 * device array of 4 MiB that each device holds from library load to the end
 * of the process. Buckets are neither split nor grouped. Flags go to the
 * device status word (mps_fp8_read_status). Calls that overlap on one device
 * share that array and race: issue them on one stream, or order them.
 * Larger inputs, and a `stream` that is capturing a graph (the descriptor
 * copy would replay from a host array that is gone), are rejected with
 * MPS_ERR_INVALID_ARGUMENT before any copy or launch.
 * No counterpart in the reference; it serves callers that cannot allocate
 * device memory in their decode loop (tight serving loops, harnesses that
 * forbid allocation). Code under graph capture launches a plan made before
 * the capture instead. */
int mps_fp8_decode_batch_noalloc(const mps_fp8_tensor *tensors, int64_t count, int64_t max_len, void *stream);

/* Capture id of `stream`: the id of the graph capture it is in, or 0 when it
 * is not capturing (hipStreamGetCaptureInfo). No counterpart in the
 * reference: the vLLM method uses it to tell a captured forward pass from an
 * eager one, so that a packed block's decoded weight is reused only within
 * one of them. */
int mps_stream_capture_id(void *stream, uint64_t *id_out);

/* Inputs of the GPU sidecar builder, all device pointers: BF16 bit patterns
 * and FP8 bytes of the same tensor (`numel` elements, shape dims[0..ndim)),
 * and the u16 scale keys (shape scale_dims[0..scale_ndim), scale_numel
 * values). */
typedef struct mps_fp8_encode_in {
  const uint16_t *bf16;
  const uint8_t *fp8;
  const uint16_t *scales;
  int64_t numel;
  int32_t ndim;
  int32_t scale_ndim;
  int64_t dims[8];
  int64_t scale_dims[8];
  int64_t scale_numel;
  int64_t max_len;           /* 1..15 (decoding needs 7) */
  int64_t threads_per_block; /* k: substreams per bucket, 1..1024 */
} mps_fp8_encode_in;

/* Build the Huffman sidecar of one tensor on the GPU, byte-identical to the
 * reference builder. Replaces huffman_cpp::huffman_build_fp8_decode_tables_entry
 * (reference kernel/build_huffman.cu:292-969, bound as
 * MPServe_cuda.huffman_build_fp8_decode_tables at kernel/wrapper.cpp:418-454),
 * which runs single-threaded on the host; same argument checks and messages.
 * Synchronises `stream` (output sizes are data dependent). The result lives in
 * device memory owned by the returned handle. */
typedef struct mps_fp8_sidecar mps_fp8_sidecar;
int mps_fp8_encode(const mps_fp8_encode_in *in, void *stream, mps_fp8_sidecar **out);
/* One AWQ int4 tensor and its sidecar, all device pointers, in either layout
 * of the reference's AWQ int4 builders (dtype views as for the FP8 tensor). */
typedef struct mps_awq_tensor {
  const uint8_t *int4;                   /* [n*m] int4 values, one per byte (low nibble) */
  const uint64_t *bitstream;             /* [bitstream_words] */
  int64_t bitstream_words;
  const uint16_t *decode_syms;           /* [num_tables,2048] */
  const uint8_t *decode_lens;            /* [num_tables,1024] packed 4-bit, 15 = ESC */
  int64_t num_tables;
  const int32_t *bucket_table;           /* [num_buckets,16] int4 value -> table id or -1 */
  const int32_t *bucket_col_start;       /* row layout: [num_buckets]; by-scale layout: NULL */
  const int32_t *bucket_col_len;         /* row layout: [num_buckets]; by-scale layout: NULL */
  const int32_t *bucket_row_offsets;     /* [num_buckets+1] bucket_row_offsets / bucket_group_offsets */
  const int32_t *row_indices;            /* [num_row_indices] row_indices / group_rows */
  int64_t num_row_indices;
  const int32_t *group_col_start;        /* by-scale layout: [num_row_indices]; row layout: NULL */
  int64_t group_size;                    /* by-scale layout: columns per group */
  const uint32_t *bucket_thread_startbit;/* [num_buckets, k+1] */
  const int64_t *bucket_bit_base;        /* [num_buckets+1] */
  int64_t num_buckets;
  int64_t k;                             /* 1..1024 */
  int64_t n, m;                          /* output shape [n, m], n*m < 2^31 */
  uint16_t *out;                         /* [n*m] BF16 bit patterns (device) */
} mps_awq_tensor;

/* Decode one AWQ int4 tensor: out[n,m] = BF16 rebuilt from int4 values + sidecar,
 * on `stream`. Replaces huffman_cpp::huffman_decode_awq_int4_bucket_entry
 * (group_col_start == NULL; reference kernel/decode_huffman.cu:877-1018 and
 * :378-475, bound at kernel/wrapper.cpp:324-369) and
 * ..._by_scale_entry (group_col_start != NULL; kernel/decode_huffman.cu:760-875
 * and :477-589, bound at kernel/wrapper.cpp:371-416). The shape/dtype checks
 * of those entries are done by the caller. max_len must be 11. Columns of a
 * row bucket are walked as e % col_len, as the builder lays them out.
 * Asynchronous: returns after the launch. */
int mps_awq_decode(const mps_awq_tensor *tensor, int64_t max_len, void *stream);

/* Batched AWQ decode plan: one launch decodes every bucket of many AWQ int4
 * tensors (either layout, mixed), largest work first. Runs of up to 1024 / k
 * consecutive buckets with identical table ids share one workgroup and its
 * tables. Creation synchronises `stream` first, then reads each tensor's
 * bucket row offsets, table ids (and column lengths) once and copies the
 * descriptors into one device allocation the plan owns (with its own status
 * word, mps_awq_plan_read_status); the pointed-to tensors must stay alive
 * while the plan is used, and a tensor whose bucket metadata is rewritten
 * needs a new plan. Decodes are asynchronous on `stream`. A launch runs one
 * workgroup per CU that takes the plan's work records from a queue in the
 * plan's memory; the plan holds 32 such queues and gives each stream that
 * launches it its own (a 33rd stream is refused with MPS_ERR_RUNTIME), so
 * launches on different streams may overlap. A graph replays with the queue
 * of the stream it was captured on.
 * No counterpart in the reference, which launches once per tensor
 * (kernel/decode_huffman.cu:857, :998). */
typedef struct mps_awq_plan mps_awq_plan;
int mps_awq_plan_create(const mps_awq_tensor *tensors, int64_t count, void *stream, mps_awq_plan **plan_out);
int mps_awq_plan_decode(mps_awq_plan *plan, void *stream);
/* Decode the plan into a buffer laid out like its outputs, moved to `out`, as
 * mps_fp8_plan_decode_into does (the move must keep 8-byte alignment); the
 * flags go to the device status word. No counterpart in the reference: it
 * serves the AWQ decode ops' per-sidecar plan cache. */
int mps_awq_plan_decode_into(mps_awq_plan *plan, uint16_t *out, void *stream);
int mps_awq_plan_info(const mps_awq_plan *plan, int64_t *work_items);
int mps_awq_plan_read_status(mps_awq_plan *plan, void *stream, uint32_t *status_out);
int mps_awq_plan_destroy(mps_awq_plan *plan);

/* Inputs of the AWQ int4 sidecar builders, all device pointers: BF16 bit
 * patterns and int4 values (one per byte, low nibble) of an [n, m] weight, and
 * the u16 (BF16 bit) scales: one value, [n] (scale_ndim 1) or block-wise
 * [n/bs0, m/bs1] (scale_ndim 2). by_scale = 0 builds row buckets, 1 builds
 * buckets of quantisation groups of one exact scale (at most group_cap each). */
typedef struct mps_awq_encode_in {
  const uint16_t *bf16;
  const uint8_t *int4;
  const uint16_t *scales;
  int64_t n, m;
  int32_t scale_ndim;
  int32_t by_scale;
  int64_t scale_dims[2];
  int64_t scale_numel;
  int64_t max_len;           /* 1..15 (decoding needs 11) */
  int64_t threads_per_block; /* k: substreams per bucket, 1..1024 */
  int64_t group_cap;         /* by_scale: groups per bucket, > 0 */
} mps_awq_encode_in;

/* Build the AWQ int4 sidecar of one weight on the GPU, byte-identical to the
 * reference builders, which run single-threaded on the host:
 *   by_scale = 0: huffman_cpp::huffman_build_awq_int4_bucket_decode_tables_entry
 *     (reference kernel/build_huffman.cu:1583-2126, bound as
 *     MPServe_cuda.huffman_build_awq_int4_bucket_decode_tables at kernel/wrapper.cpp:258-288);
 *   by_scale = 1: ..._by_scale_entry (kernel/build_huffman.cu:1075-1580, bound as
 *     MPServe_cuda.huffman_build_awq_int4_bucket_decode_tables_by_scale at kernel/wrapper.cpp:290-321).
 * Same argument checks and messages. The result uses the FP8 handle's 17
 * slots: slots 0-13 in the reference's order of the row-bucket dict (slot 3 is
 * table_qv_u16, slot 7 bucket_table_i32 [B,16]); by scale, slot 5 holds
 * bucket_group_offsets_i32, slot 6 group_rows_i32, slot 8 group_col_start_i32
 * and slot 13 shape_nmkg_i64 (slot 9 is empty). Slots 14-16 are empty. */
int mps_awq_encode(const mps_awq_encode_in *in, void *stream, mps_fp8_sidecar **out);

/* The same builds into the caller's memory, without a handle. `alloc` is asked
 * for device memory on the current device, usable on `stream`, 256-byte
 * aligned: each non-empty output once, by its slot (0..16, the handle's order),
 * and workspaces as slot -1; it returns NULL when it has none (then
 * MPS_ERR_NO_MEMORY). Called on the calling thread. sizes17 and stats4 are as
 * mps_fp8_sidecar_sizes and mps_fp8_sidecar_stats give them. The last passes may
 * still be running on `stream` after MPS_OK: the caller synchronises it before it
 * uses outputs or inputs on another stream or on the host (the Python ops do so
 * before they return), and frees workspaces in stream order. After an error the
 * stream is idle. No counterpart in the reference, whose outputs are host tensors;
 * it spares a serving or compressing program, whose allocator caches memory, the
 * builder's own device allocations and the copies out of a handle. */
typedef void *(*mps_encode_alloc)(void *ctx, int32_t slot, int64_t bytes);
int mps_fp8_encode_alloc(const mps_fp8_encode_in *in, void *stream, mps_encode_alloc alloc, void *ctx,
                         int64_t *sizes17, int64_t *stats4);
int mps_awq_encode_alloc(const mps_awq_encode_in *in, void *stream, mps_encode_alloc alloc, void *ctx,
                         int64_t *sizes17, int64_t *stats4);

/* Element counts of the 17 outputs, in the reference's order (kernel/wrapper.cpp:429-446):
 * decode_syms_u16, decode_lens_u8, table_scale_u16, table_fp8_u16, bucket_scale_u16,
 * bucket_row_offsets_i32, row_indices_i32, bucket_table_i32, bucket_col_start_i32,
 * bucket_col_len_i32, bucket_thread_startbit_u32, bucket_bit_base_i64, bitstream_u64,
 * shape_nmk_i64, bucket_U_i32, bucket_unique_gid_i32, bucket_fp8_uidx_i16. */
int mps_fp8_sidecar_sizes(const mps_fp8_sidecar *sc, int64_t *sizes17);
/* Copy the 17 outputs into caller buffers (host or device; hipMemcpyDefault); synchronises. */
int mps_fp8_sidecar_copy(const mps_fp8_sidecar *sc, void *const *dst17, void *stream);
/* {keys coded with ESC, elements equal to their key's esc_sym, distinct (key, symbol) pairs, hash slots}. */
int mps_fp8_sidecar_stats(const mps_fp8_sidecar *sc, int64_t *stats4);
int mps_fp8_sidecar_free(mps_fp8_sidecar *sc);

/* Read and clear the MPS_STATUS_* flags the single-tensor decodes
 * (mps_fp8_decode, mps_awq_decode, mps_fp8_plan_decode_into) on `device`
 * recorded since the last call. The word is per device, not per stream:
 * flags of decodes on any stream of the device accumulate in it. It is a
 * module global of the library (no allocation). Synchronises `stream` first. */
int mps_fp8_read_status(int device, void *stream, uint32_t *status_out);

/* ---------------------------------------------------------------- MXFP4 and experts
 * No counterpart in the reference, whose 4-bit weights are AWQ int4 ones. All
 * calls are asynchronous on `stream`, allocate nothing, and can be captured
 * into a graph. Workspaces are the caller's device memory, 16-byte aligned,
 * and are free again when the call's work on `stream` has ended. */

/* Element types. */
#define MPS_TYPE_BF16 0
#define MPS_TYPE_F16 1
#define MPS_TYPE_F32 2
#define MPS_TYPE_MXFP4 3 /* operands of mps_mxfp4_multiply only */

#define MPS_MAX_EXPERTS 1024

/* MXFP4 of x[rows, k] (`row_stride` elements from row to row): codes
 * [rows, 16 * ceil(k / 32)], two codes a byte, the earlier element in the low
 * half, a row's last block filled up with zero codes; scales
 * [rows, ceil(k / 32)], the byte s of 2^(s - 127). The scale is
 * 2^(floor(log2 max|x|) - 2), at least 2^-127; a code is the nearest value,
 * ties to the even code, magnitudes above 6 to 6. A block with an infinity or
 * a NaN gets scale 255 (it reads back as NaN) and zero codes. */
int mps_mxfp4_quantize(const void *x, int32_t type, int64_t rows, int64_t k, int64_t row_stride, uint8_t *codes,
                       uint8_t *scales, void *stream);
/* The values [rows, k] of MXFP4 codes, rounded to `type` (exact in BF16 and
 * FP32 except where 6 * 2^127 overflows). */
int mps_mxfp4_dequantize(const uint8_t *codes, const uint8_t *scales, int64_t rows, int64_t k, void *out, int32_t type,
                         void *stream);

/* out[rows, n] = x[rows, k] times the transpose of w[n, k], plus bias[n], with
 * w in MXFP4 and x in BF16, FP16 or MXFP4; FP32 sums, one rounding to
 * out_type. With experts > 0, w is [experts, n, k] and bias [experts, n]:
 * rows offsets[e] .. offsets[e + 1] are multiplied by expert e's weight and
 * rows from offsets[experts] on are set to zero. With `gather`, for 16-bit x
 * only, row j of the product is made of x's row order[j] / top instead of its
 * row j, of x's rows / top rows; MXFP4 x comes in the sorted order. The offsets
 * and the order are mps_expert_sort's (or hold its promises: offsets rise
 * from 0 to at most rows, the order's entries are below the rows of x times
 * top). Codes are 16-byte aligned; those past column k in a row's last block
 * are zero, as mps_mxfp4_quantize writes them. No workspace is needed for MXFP4
 * x, nor for 16-bit x whose rows are whole blocks at 16-byte addresses. */
typedef struct mps_mxfp4_product {
  const void *x;           /* [rows, k] with x_stride, or MXFP4 codes */
  const uint8_t *x_scales; /* MXFP4 only */
  int64_t x_stride;        /* elements from row to row; unused for MXFP4 */
  const uint8_t *w;
  const uint8_t *w_scales;
  const void *bias; /* may be NULL */
  void *out;
  const int32_t *offsets; /* [experts + 1] */
  const int32_t *order;   /* [rows], gather only */
  int64_t rows, n, k;
  int64_t experts; /* 0: one weight for all rows */
  int64_t top;
  int32_t gather;
  int32_t x_type, bias_type, out_type;
} mps_mxfp4_product;
int mps_mxfp4_product_workspace(const mps_mxfp4_product *product, int64_t *bytes);
int mps_mxfp4_multiply(const mps_mxfp4_product *product, void *workspace, int64_t workspace_bytes, void *stream);

/* Sort the pairs of tokens and experts: ids[tokens, top] (int32, or int64 with
 * ids_64) names each pair's expert; a pair whose id is not in [0, experts) has
 * none. Pairs are ordered by expert, those of an expert as they come, those
 * of none last: order[j] is the pair (token * top + slot) at place j,
 * positions[pair] its place, -1 for a pair of no expert, and
 * offsets[0 .. experts] where each expert's pairs begin and the last one's end. */
int mps_expert_sort_workspace(int64_t tokens, int64_t top, int64_t experts, int64_t *bytes);
int mps_expert_sort(const void *ids, int32_t ids_64, int64_t tokens, int64_t top, int64_t experts, int32_t *order,
                    int32_t *positions, int32_t *offsets, void *workspace, int64_t workspace_bytes, void *stream);
/* rows[tokens * top, width]: x's row t at the place of each of its pairs; rows
 * from offsets[experts] on are zero. */
int mps_expert_gather(const void *x, int32_t type, int64_t tokens, int64_t top, int64_t experts, int64_t width,
                      const int32_t *order, const int32_t *positions, const int32_t *offsets, void *rows, void *stream);
/* out[tokens, width]: row t is the sum over its pairs' places p of
 * weights[pair] * y[p] (weights NULL: of y[p]), in FP32 and in the pairs'
 * order, without the pairs of no expert. Also the gradient of the gather. */
int mps_expert_combine(const void *y, int32_t type, const void *weights, int32_t weights_type, int64_t tokens,
                       int64_t top, int64_t width, const int32_t *positions, void *out, void *stream);
/* Gradients of mps_expert_combine: dy[j] = weights[pair] * dout[token] and
 * dweights[pair] = <y[j], dout[token]> for the pair at place j; zero for the
 * pairs of no expert. dy or dweights may be NULL, if that gradient is not
 * wanted; y may be NULL without dweights. */
int mps_expert_combine_grad(const void *y, const void *dout, int32_t type, const void *weights, int32_t weights_type,
                            int64_t tokens, int64_t top, int64_t experts, int64_t width, const int32_t *order,
                            const int32_t *positions, const int32_t *offsets, void *dy, void *dweights, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* MPSERVE_AMD_H */
