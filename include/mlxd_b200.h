/*
 * C ABI of the B200 image-transform-and-batch library (libmlxd_b200.so).
 *
 * mlx-data has no C ABI of its own: its boundary for this path is a set of C++
 * virtuals (op::ImageTransformOp::apply_image, stream::Batch::next,
 * core::merge_batch).  The entry points below are what those virtuals bind to
 * when the path runs on the GPU; each one names the reference interface it
 * replaces.  Plain pointers and sizes only, an int status on every call, no
 * exceptions and no C++ or torch types cross this boundary.
 *
 * Images are [H, W, C] uint8, C-contiguous (mlx/data/core/image/Image.h:35-49),
 * 1 <= C <= 4.  A batch is [N, slot_h, slot_w, C_out], C-contiguous.
 */
#ifndef MLXD_B200_H
#define MLXD_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MLXD_API __attribute__((visibility("default")))

typedef struct mlxd_ctx mlxd_ctx;

enum mlxd_status {
  MLXD_OK = 0,
  MLXD_ERR_INVALID = 1,     /* bad argument; mlxd_last_error() says which */
  MLXD_ERR_CUDA = 2,        /* a CUDA call failed; message carries its text */
  MLXD_ERR_NOMEM = 3,       /* host or device allocation failed */
  MLXD_ERR_TIMEOUT = 4,     /* mlxd_batch_wait ran out of time; work still queued */
  MLXD_ERR_UNSUPPORTED = 5, /* a shape the device code cannot run (kept for callers; nothing returns it now) */
  MLXD_ERR_DEVICE = 6       /* the kernel recorded a failed self-check */
};

enum mlxd_geom {
  MLXD_GEOM_NONE = 0,
  MLXD_GEOM_RESIZE = 1, /* core::image::resize, mlx/data/core/image/ImageTransform.cpp:41-62 */
  MLXD_GEOM_AFFINE = 2  /* core::image::affine, mlx/data/core/image/ImageTransform.cpp:75-111 */
};

/* Batches are MLXD_U8 or MLXD_F32; the attention operators at the end take the others. */
enum mlxd_dtype { MLXD_U8 = 0, MLXD_F32 = 1, MLXD_BF16 = 2, MLXD_F16 = 3, MLXD_I32 = 4, MLXD_I64 = 5 };
enum mlxd_mem { MLXD_MEM_HOST = 0, MLXD_MEM_DEVICE = 1 };

/*
 * One sample's op chain, already reduced by the caller to the canonical order
 *   source -> window+mirror -> one geometric op -> window+mirror -> [gray] -> slot.
 * It stands for a run of op::ImageTransformOp::apply_image calls
 * (mlx/data/op/ImageTransform.cpp:78-369) on one key of one sample:
 *   pre_*   crops (core::image::crop, ImageTransform.cpp:64-73) and horizontal
 *           flips (core::image::hflip, :123-140) that come before the geometric op;
 *   geom    image_resize / image_resize_smallest_side (target size in geom_w,
 *           geom_h) or image_rotate (matrix in mx, output size in geom_w, geom_h,
 *           both computed by the caller exactly as :80-86 and :113-121 do);
 *   post_*  crops and flips after it.
 * With geom == NONE the geometric output is the pre window itself and
 * geom_w, geom_h must equal pre_w, pre_h.  Random parameters (crop rectangles,
 * flip decisions) are drawn by the caller on the host.
 *
 * Resize with 4 channels: the reference passes the channel count to its resize
 * library as the pixel layout (ImageTransform.cpp:49-58), and layout 4 is
 * RGBA, whose colour channels are weighted by alpha while filtering.  The
 * kernels behind this struct filter every channel independently, also for
 * C == 4, so a 4-channel resize differs from the reference wherever alpha
 * varies.  The pipeline layer above this ABI refuses such resizes unless the
 * caller opted in; at this level the caller is expected to know.
 */
typedef struct mlxd_sample_desc {
  const uint8_t* src; /* [src_h, src_w, C]; device memory is read in the aligned 16-byte units that hold its bytes */
  int32_t src_h, src_w;
  int32_t pre_x, pre_y, pre_w, pre_h;
  int32_t pre_flip;
  int32_t geom;
  int32_t geom_w, geom_h;
  float mx[6];
  int32_t post_x, post_y, post_w, post_h;
  int32_t post_flip;
  int32_t reserved;
} mlxd_sample_desc;

/*
 * The batch the samples are written into: array::batch
 * (mlx/data/Array.cpp:465-498) with core::BatchShape (mlx/data/core/BatchShape.cpp:26-45)
 * followed by the cast that reference pipelines run as a Python lambda
 * (README.md:55-57): x.astype(float32) / 255, optionally (x/255 - mean) / std.
 * Sample i occupies slot i; its post window sits in the slot's top-left corner
 * and the rest of the slot holds the pad value (cast like every other pixel).
 */
typedef struct mlxd_batch_desc {
  void* dst;           /* [n, slot_h, slot_w, C_out] of out_dtype */
  int32_t slot_h, slot_w;
  int32_t channels;    /* C of every source image */
  int32_t gray;        /* 1: core::image::channel_reduction (ImageTransform.cpp:142-182) after the post window; C_out = 1 */
  int32_t gray_m[3];   /* its 16.16 fixed-point multipliers, (int)(coef * 65536) */
  int32_t gray_bias;   /* (int)(bias * 65536) */
  int32_t out_dtype;   /* MLXD_U8: raw bytes; MLXD_F32: cast below */
  int32_t normalise;   /* 0: x / divisor; 1: (x / divisor - mean[c]) / std[c] */
  float divisor;       /* 255 for the usual cast; 1 gives a plain astype */
  float mean[4];
  float std_[4];
  double pad_value;    /* batch pad value, converted to uint8 like Array::fill (mlx/data/Array.cpp:123-134) */
  int32_t src_mem;     /* mlxd_mem of every sample's src */
  int32_t dst_mem;     /* mlxd_mem of dst */
} mlxd_batch_desc;

typedef struct mlxd_stats {
  uint64_t batches;        /* fused launches issued */
  uint64_t samples;
  uint64_t kernel_launches;
  uint64_t h2d_bytes;
  uint64_t d2h_bytes;
  uint64_t device_bytes_reserved; /* staging + output arenas currently held */
  uint64_t kernel_ns;             /* summed device time of the timed launches (CUDA events around each kernel) */
  uint64_t timed_launches;        /* launches included in kernel_ns; 0 unless timing is on */
  uint64_t algo_src_bytes;        /* summed source footprints: the uint8 source rectangle each sample's chain can read */
  uint64_t algo_dst_bytes;        /* summed batch tensor bytes written, padding included */
  uint64_t h2d_ns;                /* timed launches: device time of the host-to-device stage (gather kernel or copies,
                                   * from the first of a batch's parts where those go out while the rest is packed) */
  uint64_t d2h_ns;                /* timed launches: device time of the batch's copy back to the host */
  uint64_t host_stage_ns;         /* host time spent copying sources from ordinary memory into page-locked blocks */
} mlxd_stats;

/* Context: one device, n_lanes independent lanes.  A lane owns a CUDA stream, a
 * device staging arena and an output arena; calls on one lane are stream
 * ordered, different lanes overlap.  Replaces the role of core::ThreadPool
 * workers under stream::Prefetch (mlx/data/stream/Prefetch.cpp:29-56): one
 * prefetch worker drives one lane. */
MLXD_API int mlxd_ctx_create(int device, int n_lanes, mlxd_ctx** out);
MLXD_API void mlxd_ctx_destroy(mlxd_ctx* ctx);

/* Text of the last error raised on the calling thread. */
MLXD_API const char* mlxd_last_error(void);

/* Page-locked host memory for sample and batch storage; backs Array storage
 * through the external-storage constructor (mlx/data/Array.h:28-31).  The
 * blocks are mapped into the GPU's address space and remembered: when every
 * source of a host-fed mlxd_fused_batch lies in such blocks, a kernel reads
 * just the rectangle each chain needs over the bus (for a centre crop of a
 * 1080 x 1920 frame that is 57 % of the bytes a row-contiguous copy moves);
 * page-locked memory that did not come from here goes through the copy engines,
 * and sources in ordinary (pageable) memory are first packed - needed rectangle
 * only - into a page-locked block of the lane by the calling thread and up to
 * MLXD_PACK_THREADS - 1 helpers (default 4 threads in all) and copied, large
 * batches in parts while the rest is being packed.  MLXD_HOST_GATHER=0 in the environment turns the kernel path off. */
MLXD_API void* mlxd_pinned_alloc(size_t bytes);
MLXD_API void mlxd_pinned_free(void* p);

/* PCI address of a CUDA device as "dddd:bb:dd.f" (NUL-terminated, len >= 16):
 * the name of its directory under /sys/bus/pci/devices, where a host finds the
 * NUMA node its loader threads and page-locked pools belong on.  (No
 * counterpart in the reference.) */
MLXD_API int mlxd_device_pci_bus_id(int device, char* out, size_t len);

/* Device memory on the context's GPU, for sources and batches that stay in
 * HBM (no counterpart in the reference, which is host-only).  NULL on failure. */
MLXD_API void* mlxd_device_alloc(mlxd_ctx* ctx, size_t bytes);
MLXD_API void mlxd_device_free(mlxd_ctx* ctx, void* p);

/* Bracket every fused kernel with CUDA events on the stream it is launched on
 * and add the elapsed device time to mlxd_stats.kernel_ns (off by default). */
MLXD_API int mlxd_ctx_set_timing(mlxd_ctx* ctx, int on);

/* The fused batch for callers that cannot allocate.  It has no counterpart in
 * the reference.  Who needs it: a loader plug-in that runs inside a training
 * step whose framework has handed the whole GPU to its own memory pool, a
 * service that bans allocator calls once it is warm, a process sitting at its
 * memory limit - for them a cudaMalloc (or a pinned-host allocation) in the
 * data path is a failure or a stall, and the other entry points do allocate:
 * descriptor tables, the cast table and a status word, on demand.  Here those
 * live in a fixed array inside the library image, so the call allocates
 * nothing on the device or the host, and needs no context.
 *
 * Same meaning as mlxd_fused_batch_on_stream: sources and destination are
 * device memory (batch->src_mem == batch->dst_mem == MLXD_MEM_DEVICE), the
 * kernel is queued on the caller's CUDA stream, the descriptors are read
 * before the call returns.  Limits and rules:
 *  - at most MLXD_NOALLOC_MAX_SAMPLES samples per call; more is refused with
 *    MLXD_ERR_INVALID (split the batch, or use the allocating entry point);
 *  - the array (about 0.15 MB) is held by every GPU that loads the library
 *    until the process exits;
 *  - the first call on a device looks up the array's device address; make
 *    that first call before any stream capture;
 *  - every call waits on the host until the stream has drained (its small
 *    tables are copied from fixed host storage that the next call reuses), so
 *    the host blocks behind whatever is queued on that stream before it;
 *  - the stream must belong to `device`; the calling thread's current device
 *    is the same after the call as before it;
 *  - all calls share the one array, which keeps the previous call's contents
 *    (the call clears what must start at zero): two calls whose kernels can
 *    overlap on the GPU - different streams, or different host threads - race;
 *    order them on one stream;
 *  - the kernel's self-check word (a resize chunk beyond its planned shared
 *    memory) is read back at the start of the NEXT call on the same stream,
 *    which then returns MLXD_ERR_DEVICE and launches nothing; after the last
 *    call of a run ask mlxd_noalloc_status. */
#define MLXD_NOALLOC_MAX_SAMPLES 1024
MLXD_API int mlxd_fused_batch_noalloc(
    int device, void* cuda_stream, const mlxd_sample_desc* samples, int n, const mlxd_batch_desc* batch);

/* Self-check word of the most recent mlxd_fused_batch_noalloc kernel on this
 * device, read from the same fixed array (no allocation; no counterpart in the
 * reference).  Waits for `cuda_stream`, stores the word in *status (0 = clean),
 * clears it, and returns MLXD_ERR_DEVICE when it was set. */
MLXD_API int mlxd_noalloc_status(int device, void* cuda_stream, int32_t* status);

/* Enqueue one fused batch on a lane and return: host sources are copied to the
 * device (only the rows the chain reads), one kernel writes every slot, and a
 * host dst is copied back.  Replaces stream::Batch::next -> core::merge_batch
 * (mlx/data/stream/Batch.cpp:25-39, mlx/data/core/Utils.cpp:209-252) together
 * with the per-sample op calls listed at mlxd_sample_desc.  Host memory must
 * stay untouched until mlxd_batch_wait returns MLXD_OK. */
MLXD_API int mlxd_fused_batch(
    mlxd_ctx* ctx, int lane, const mlxd_sample_desc* samples, int n, const mlxd_batch_desc* batch);

/* Wait for everything queued on a lane, at most timeout_ms (< 0: no limit).
 * Replaces future.get() in stream::Prefetch::next (mlx/data/stream/Prefetch.cpp:43-53). */
MLXD_API int mlxd_batch_wait(mlxd_ctx* ctx, int lane, int timeout_ms);

/* Same work for device-resident sources and destination, launched on the
 * caller's CUDA stream (a cudaStream_t passed as void*; NULL is the default
 * stream).  Nothing is copied except the descriptors (those of up to 128 samples
 * travel with the launch, unless a resize among them runs in one of the kernels for strong
 * shrinks).
 *
 * A stream under capture gets the call as nodes of the graph: the descriptors become
 * the graph's own, in an allocation node, so such a graph follows the rules of graphs
 * with memory nodes (one instance at a time, no child graph).  A replay reads the
 * sources and writes the destination given here, and sets the self-check word of this
 * context, which therefore has to outlive the graph; it is not timed. */
MLXD_API int mlxd_fused_batch_on_stream(
    mlxd_ctx* ctx, void* cuda_stream, const mlxd_sample_desc* samples, int n, const mlxd_batch_desc* batch);

/* Self-check word of the kernels launched by mlxd_fused_batch_on_stream: waits
 * for `cuda_stream`, stores the word in *status (0 = clean; 8: a resize chunk with
 * more source rows or bytes than planned, whose rows were then not written), clears
 * it, and returns MLXD_ERR_DEVICE when it was set.  The lanes of mlxd_fused_batch report the
 * same word through mlxd_batch_wait.  No counterpart in the reference, whose
 * CPU ops throw where they stand. */
MLXD_API int mlxd_stream_status(mlxd_ctx* ctx, void* cuda_stream, int32_t* status);

/* One entry per named op, host buffers in and out, synchronous; for chains
 * that cannot be fused (a host callback between two ops).  Each runs the same
 * kernel with a one-stage program. */
/* core::image::resize, mlx/data/core/image/ImageTransform.cpp:41-62
 * (c == 4: channels filtered independently, see mlxd_sample_desc) */
MLXD_API int mlxd_image_resize(
    mlxd_ctx* ctx, const uint8_t* src, int h, int w, int c, uint8_t* dst, int dh, int dw);
/* core::image::crop, mlx/data/core/image/ImageTransform.cpp:64-73 */
MLXD_API int mlxd_image_crop(
    mlxd_ctx* ctx, const uint8_t* src, int h, int w, int c, int x, int y, int cw, int ch, uint8_t* dst);
/* core::image::hflip, mlx/data/core/image/ImageTransform.cpp:123-140 */
MLXD_API int mlxd_image_hflip(mlxd_ctx* ctx, const uint8_t* src, int h, int w, int c, uint8_t* dst);
/* core::image::affine, mlx/data/core/image/ImageTransform.cpp:75-111; th, tw as computed at :80-86 */
MLXD_API int mlxd_image_affine(
    mlxd_ctx* ctx, const uint8_t* src, int h, int w, int c, const float mx[6], int th, int tw, uint8_t* dst);
/* core::image::channel_reduction, mlx/data/core/image/ImageTransform.cpp:142-182 */
MLXD_API int mlxd_image_channel_reduction(
    mlxd_ctx* ctx, const uint8_t* src, int h, int w, const int32_t m_fixed[3], int32_t bias_fixed, uint8_t* dst);
/* array::batch for uint8 images, mlx/data/Array.cpp:465-498 */
MLXD_API int mlxd_batch_pad(
    mlxd_ctx* ctx, const uint8_t* const* srcs, const int32_t* hs, const int32_t* ws, int n, int c,
    int slot_h, int slot_w, double pad_value, uint8_t* dst);
/* the float32 cast of README.md:55-57; count pixels of c channels */
MLXD_API int mlxd_cast_scale_normalise(
    mlxd_ctx* ctx, const uint8_t* src, int64_t count, int c, float divisor,
    const float* mean, const float* std_, float* dst);

MLXD_API int mlxd_stats_get(mlxd_ctx* ctx, mlxd_stats* out);

/* ---- attention over batches of images and clips ----------------------------
 * What a model does with a batch once its patches are projected: queries and
 * keys are turned by where a patch lies (time, row, column), normalised per
 * head, and text reads the images.  The reference stops at the batch and has
 * no counterpart.  All memory is device memory of `device`; everything is
 * queued on the caller's CUDA stream (NULL: the default stream) and may be
 * captured into a graph.  Nothing is allocated: the calls that need scratch
 * memory take a workspace, whose contents matter only during the call.  The
 * structs are read before the call returns; a pointer that is not aligned to
 * its elements (a workspace: to 16 bytes) is refused.  Results do not depend on the
 * order in which blocks run: there are no atomic sums. */

/* A [batch, tokens, heads, head_dim] tensor, head_dim contiguous, the other
 * strides in elements and free (views of a joint projection, for instance). */
typedef struct mlxd_heads {
  void* data;
  int64_t stride_batch, stride_token, stride_head;
} mlxd_heads;

#define MLXD_ROTARY_MAX_AXES 4
#define MLXD_ROTARY_MAX_HEAD_DIM 256

/* Rotary positions with several axes.  The pairs of a head are dealt to the
 * axes: sections[a] pairs to axis a, in order (interleaved == 0) or one in
 * turn to every axis that has some left (interleaved == 1).  Pair i turns by
 * the angle float32(position of its axis) * frequencies[i], a float32 product;
 * (x, y) -> (x cos - y sin, y cos + x sin), inverse: the other way round, which
 * is the gradient too.  Pairs are (i, i + P), or (2i, 2i + 1) if `adjacent`, with
 * P = the sum of the sections; elements from 2P on pass through unturned.
 *
 * k may be absent (k_heads == 0).  q_out and k_out may be q and k themselves
 * (same pointer, same strides); other overlaps are not allowed. */
typedef struct mlxd_rotary_desc {
  int32_t dtype;                 /* of q, k and their results: MLXD_F32, MLXD_BF16 or MLXD_F16 */
  int32_t batch, tokens, q_heads, k_heads;   /* at most 2^29 heads */
  int32_t head_dim;              /* even, at most MLXD_ROTARY_MAX_HEAD_DIM */
  mlxd_heads q, k, q_out, k_out;
  const void* positions;         /* [n_axes, batch, tokens] */
  int32_t positions_dtype;       /* MLXD_I32, MLXD_I64 or MLXD_F32 */
  int64_t positions_stride_axis, positions_stride_batch, positions_stride_token;
  const float* frequencies;      /* [P] */
  int32_t n_axes;
  int32_t sections[MLXD_ROTARY_MAX_AXES];
  int32_t adjacent, interleaved, inverse;
  /* the norm in the same pass (mlxd_qk_norm_rotary and its backward): x / sqrt(mean(x^2) + eps) * weight for each head,
   * ahead of the rotation */
  const void* q_weight;          /* [head_dim], NULL: all ones */
  const void* k_weight;
  int32_t weight_dtype;          /* MLXD_F32, MLXD_BF16 or MLXD_F16 */
  float eps;
  /* backward only: the gradients of the results come in here; those of q and k leave in q_out and k_out */
  mlxd_heads q_grad, k_grad;
  void* q_weight_grad;           /* [head_dim] of weight_dtype, NULL where the weight is */
  void* k_weight_grad;
  void* workspace;               /* mlxd_qk_norm_rotary_workspace bytes, 16-byte aligned */
  size_t workspace_bytes;
} mlxd_rotary_desc;

MLXD_API int mlxd_rotary(int device, void* cuda_stream, const mlxd_rotary_desc* d);
MLXD_API int mlxd_qk_norm_rotary(int device, void* cuda_stream, const mlxd_rotary_desc* d);
/* Bytes that the backward pass needs for the sums of the weights' gradients. */
MLXD_API int mlxd_qk_norm_rotary_workspace(int device, const mlxd_rotary_desc* d, size_t* bytes);
MLXD_API int mlxd_qk_norm_rotary_backward(int device, void* cuda_stream, const mlxd_rotary_desc* d);

#define MLXD_CROSS_MAX_HEAD_DIM 128

/* Cross attention: softmax(scale * q k^T) v, q of `q_tokens` and k, v of
 * `kv_tokens` tokens; query head h reads key head h / (q_heads / kv_heads).
 * Sample b reads its first lengths[b] keys (NULL: all; values outside
 * 0..kv_tokens are taken as the nearest of them), of these the ones whose byte
 * in key_mask [batch, kv_tokens] is not 0 (NULL: all).  What lies in k and v
 * where nothing is read has no effect, whatever it is.  A sample with no key
 * to read gets zeros, -infinity in lse, and gradients of zero; a row whose
 * scores are all -infinity has no weights in either pass.  What is not a number in q, or in a key or
 * value that is read, makes the rows that read it NaN, and their lse where it
 * is in a score.
 *
 * The weights P and, in the backward pass, dS = P (dP - delta) are rounded to
 * `dtype`, as operands of the products; sums are float32.
 *
 * lse [batch, q_heads, q_tokens] float32 is the natural logarithm of each
 * row's sum of exponentials; NULL where no backward pass follows. */
typedef struct mlxd_cross_desc {
  int32_t dtype;                 /* of every tensor here: MLXD_BF16 or MLXD_F16 */
  int32_t batch, q_tokens, kv_tokens, q_heads, kv_heads;
  int32_t head_dim;              /* a multiple of 8, at most MLXD_CROSS_MAX_HEAD_DIM */
  float scale;                   /* positive */
  mlxd_heads q, k, v, out;       /* data 16-byte aligned, strides multiples of 8 */
  float* lse;
  const void* lengths;
  int32_t lengths_dtype;         /* MLXD_I32 or MLXD_I64 */
  const uint8_t* key_mask;
  int64_t key_mask_stride;       /* between two samples */
  /* backward only: out and lse as the forward pass left them */
  mlxd_heads dout, dq, dk, dv;
  void* workspace;               /* mlxd_cross_attention_workspace bytes, 16-byte aligned */
  size_t workspace_bytes;
} mlxd_cross_desc;

MLXD_API int mlxd_cross_attention_workspace(int device, const mlxd_cross_desc* d, int backward, size_t* bytes);
MLXD_API int mlxd_cross_attention(int device, void* cuda_stream, const mlxd_cross_desc* d);
MLXD_API int mlxd_cross_attention_backward(int device, void* cuda_stream, const mlxd_cross_desc* d);
/* The same where lse has a gradient too: lse_grad [batch, q_heads, q_tokens] float32, NULL for none. */
MLXD_API int mlxd_cross_attention_backward_lse(int device, void* cuda_stream, const mlxd_cross_desc* d, const float* lse_grad);

/* Self-check word of the kernels of cross attention on this device: waits for `cuda_stream`, stores the word in *status
 * (0 = clean; 1: a kernel gave up waiting for its own copies or products, which none does unless the device is at fault)
 * and returns MLXD_ERR_DEVICE when it is set.  The word is one for all streams of the device and stays set for the life of
 * the process.  The rows that such a kernel was to write hold NaN.  Not under capture. */
MLXD_API int mlxd_attention_status(int device, void* cuda_stream, int32_t* status);

#ifdef __cplusplus
}
#endif
#endif /* MLXD_B200_H */
