/*
 * merv_hip.h -- C ABI of libmerv_hip.so: the MI355X (gfx950) implementation of MERV's multi-encoder video
 * forward path (four visual encoders -> 3davg+linear projectors -> cross-encoder fusion -> BOS splice),
 * plus the bit-exact frame-index sampler.
 *
 * The reference (princetonvisualai/merv) is pure Python; there is no FFI in it. Each entry point below
 * therefore names the Python call it replaces (file:line under /root/reference) -- that call is what a
 * maintainer re-points at this library (see INTEGRATION.md for the ctypes stubs).
 *
 * Conventions
 *  - Plain pointers and sizes only. Every device buffer (pixels, weights, workspace, outputs) is owned by the
 *    caller (PyTorch allocator); the library owns only host-side descriptors.
 *  - All device work is enqueued on the caller's hipStream_t (passed as void*) and is asynchronous; nothing
 *    here synchronises the device or allocates device memory, so every call is hipGraph-capturable.
 *  - Return value: 0 = ok, non-zero = error; merv_last_error() gives a thread-local message. No exceptions
 *    cross the ABI.
 *  - Activations and GEMM weights are bf16 (raw uint16 bits); biases, LayerNorm / LayerScale parameters,
 *    temporal embeddings and the fusion vector are fp32.
 */
#ifndef MERV_HIP_H
#define MERV_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* 2 (round 3): kernel-level profiler classes 5-12 added to merv_prof_*; every round-2 entry point unchanged
 * 3 (round 5): the two opt-in one-launch decode forms (merv_decode_attn_oproj*, merv_decode_chain*: measured slower, EXPERIMENTS.md
 *    section 5) are no longer exported; every other entry point unchanged
 * 4 (round 6): merv_tuning_hooks, merv_debug_gemm_mxfp8_forms, merv_debug_set_rest_fork, merv_decode_sample_advance,
 *    merv_decode_attention_split_prefetch and merv_encoder_set_latency_critical added; the product build reads no environment variable and
 *    merv_debug_set_* are no-ops in it */
#define MERV_ABI_VERSION 4

/* activation kinds */
enum { MERV_ACT_NONE = 0, MERV_ACT_GELU_ERF = 1, MERV_ACT_GELU_TANH = 2, MERV_ACT_QUICK_GELU = 3 };
/* pixel layouts */
enum { MERV_PIX_BFCHW = 0 /* [B,F,3,H,W]: DINOv2, SigLIP, ViViT */, MERV_PIX_BCFHW = 1 /* [B,3,F,H,W]: LanguageBind */ };
/* pixel dtypes */
enum { MERV_DT_F32 = 0, MERV_DT_BF16 = 1 };

/* Geometry / semantics of one visual encoder (SURVEY.md Appendix A lists the four instances). */
typedef struct merv_encoder_desc {
    int32_t dim;            /* embed dim D (1024 / 768) */
    int32_t heads;          /* D / 64 */
    int32_t mlp_dim;        /* 4096 / 3072 */
    int32_t layers;         /* number of blocks actually run (23 / 23 / 12 / 11 for merv-full) */
    int32_t patch;          /* spatial patch size (14 / 16) */
    int32_t tubelet;        /* temporal patch size (2 for ViViT, else 1) */
    int32_t img;            /* 224 */
    int32_t frames;         /* input frames per video (16 / 16 / 32 / 16) */
    int32_t pix_layout;     /* MERV_PIX_* */
    int32_t prefix_tokens;  /* cls (+ register) tokens per sequence (1 / 5 / 1 / 0) */
    int32_t joint_space_time; /* 1: one sequence per video over all tubelets (ViViT); 0: one per frame */
    int32_t pre_ln;         /* LayerNorm right after the embeddings (LanguageBind pre_layrnorm) */
    int32_t final_ln;       /* LayerNorm applied to the selected output (ViViT) */
    int32_t layerscale;     /* LayerScale on both residual branches (DINOv2) */
    int32_t temporal_frames;/* >0: temporal-attention sub-block over this many frames (LanguageBind: 8) */
    int32_t act;            /* MERV_ACT_* of the MLP */
    int32_t k_pad;          /* patch-embedding K padded to a multiple of 64 (588 -> 640) */
    float ln_eps;
} merv_encoder_desc;

/* Per-block parameters. GEMM weights are nn.Linear-layout [out, in] bf16; q/k/v are concatenated row-wise. */
typedef struct merv_layer_weights {
    const float *ln1_w, *ln1_b;
    const void *qkv_w;  const float *qkv_b;     /* [3D, D], [3D] */
    const void *proj_w; const float *proj_b;    /* [D, D], [D] */
    const float *ls1;                           /* [D] or NULL */
    const float *ln2_w, *ln2_b;
    const void *fc1_w;  const float *fc1_b;     /* [mlp, D] */
    const void *fc2_w;  const float *fc2_b;     /* [D, mlp] */
    const float *ls2;                           /* [D] or NULL */
    /* temporal sub-block (LanguageBind, modeling_video.py:133-155); NULL otherwise */
    const float *t_emb;                         /* [t, D] */
    const float *t_ln_w, *t_ln_b;
    const void *t_qkv_w; const float *t_qkv_b;
    const void *t_proj_w; const float *t_proj_b;
} merv_layer_weights;

typedef struct merv_encoder_weights {
    const void *patch_w;     /* [D, k_pad] bf16, conv kernel flattened (c, dt, dy, dx), zero padded */
    const float *patch_b;    /* [D] or NULL (LanguageBind conv has no bias) */
    const void *prefix;      /* [prefix_tokens, D] bf16: cls (+pos) / register rows, or NULL */
    const void *pos;         /* [patches per sequence, D] bf16 position embedding of the patch tokens */
    const float *pre_ln_w, *pre_ln_b;
    const float *final_ln_w, *final_ln_b;
    const merv_layer_weights *layers; /* [desc.layers] (host array, copied at create) */
} merv_encoder_weights;

typedef struct merv_encoder merv_encoder; /* opaque */

/* Thread-local message for the last failing call on this thread. */
const char *merv_last_error(void);
int merv_abi_version(void);

/*
 * Frame-index sampler. Replaces the np.linspace(..., dtype=int) selection in
 * merv/preprocessing/datasets/datasets.py:131-141 (and the NaN guards :46-52). Host-only, float64, bit-exact.
 *   end_frame < 0  : ids = linspace(clip_start*fps, min(N-1, clip_end*fps - 1), n); clip_end_sec NaN = "None"
 *   end_frame >= 0 : ids = linspace(0, min(N-1, end_frame), n)
 */
int merv_frame_indices(int64_t video_num_frames, double avg_fps, double clip_start_sec, double clip_end_sec,
                       int64_t end_frame, int32_t num_frames, int64_t *out_ids);

/* Per-encoder temporal subsample video[:: max_nf // nf] (merv.py:803-806). Returns count via *out_n. */
int merv_temporal_subsample(int32_t loaded_frames, int32_t max_nf, int32_t nf, int32_t *out_idx, int32_t *out_n);

/* Encoder lifecycle. Weight pointers are captured (not copied); they must outlive the encoder. */
int merv_encoder_create(const merv_encoder_desc *desc, const merv_encoder_weights *w, merv_encoder **out);
void merv_encoder_destroy(merv_encoder *enc);
size_t merv_encoder_workspace_bytes(const merv_encoder *enc, int32_t batch);
int32_t merv_encoder_num_patches(const merv_encoder *enc);   /* tokens returned per video */

/*
 * VideoBackbone.forward (languagebind/__init__.py:79-103, dinov2_video.py:132-154, vivit.py:100-118,
 * siglip.py:142-151): pixels -> [B, num_patches, D] bf16 patch tokens (second-to-last block / final-LN rule per
 * encoder, prefix tokens stripped).
 */
int merv_encoder_forward(const merv_encoder *enc, const void *pixels, int32_t pix_dtype, int32_t batch,
                         void *out_tokens, void *workspace, size_t workspace_bytes, void *stream);

/*
 * The same forward over `frames` frames per video instead of the descriptor's count: a frame-range work unit of the
 * multi-GPU placement (DINOv2 / SigLIP frames are independent sequences, dinov2_video.py:135-136,
 * siglip.py:146-147; LanguageBind clips of `temporal_frames` frames are independent by construction,
 * languagebind/video/modeling_video.py:140-146). pixels hold exactly `frames` frames per video in the encoder's layout;
 * out_tokens is [B, frames/tubelet * S, D]. frames must be a multiple of the tubelet and of temporal_frames; a joint
 * space-time encoder (ViViT) only accepts its own frame count. Workspace: merv_encoder_workspace_bytes(enc, batch) suffices
 * for any frames <= the descriptor's.
 */
int merv_encoder_forward_frames(const merv_encoder *enc, const void *pixels, int32_t pix_dtype, int32_t batch,
                                int32_t frames, void *out_tokens, void *workspace, size_t workspace_bytes, void *stream);

/*
 * The same forward with the token selection spelled out. MERV_OUT_PATCHES: what merv_encoder_forward returns (prefix tokens
 * stripped). MERV_OUT_ALL: every token of every sequence, prefix tokens first -- [B, frames/tubelet, prefix + S, D] for
 * per-frame encoders, [B, prefix + T*S, D] for a joint space-time encoder -- for the registry's other token selections
 * (merv/models/materialize.py:31-73: `classemb`, `average`, `classemb-at-first`, `all-token-with-cls`, `cls-token`, ...:
 * languagebind/__init__.py:88-98, dinov2_video.py:140-151, vivit.py:106-118), which are views / means of this tensor.
 */
#define MERV_OUT_PATCHES 0
#define MERV_OUT_ALL 1
int merv_encoder_forward_select(const merv_encoder *enc, const void *pixels, int32_t pix_dtype, int32_t batch, int32_t frames,
                                int32_t select, void *out_tokens, void *workspace, size_t workspace_bytes, void *stream);
/* out[g] = bf16(mean over r < rows of x[g * group_stride_rows + r]) (fp32 accumulation: torch.mean of a bf16 tensor), rows of D */
int merv_mean_rows(const void *x, void *out, int32_t groups, int32_t rows, int32_t D, int64_t group_stride_rows, void *stream);

/*
 * AveragePooling3DProjector.forward with mlp_type="linear" (merv/util/nn_utils.py:320-330, :31-32):
 * tokens [B, T*S*S, C] -> AdaptiveAvgPool3d((T, out_size, out_size)) -> Linear(C -> llm_dim) -> [B, T*out^2, llm_dim].
 * pooled_ws: scratch of B*T*out^2*C bf16.
 */
int merv_projector_forward(const void *tokens, int32_t batch, int32_t T, int32_t S, int32_t C, int32_t out_size,
                           const void *proj_w, const float *proj_b, int32_t llm_dim, void *pooled_ws, void *out,
                           void *stream);

/*
 * CrossAttentionAdapterLearnableQuery.forward, averagetoken=True (merv/util/nn_utils.py:487-521).
 * v[e]: [B, T, C] bf16; u = Wk^T (Wq Q + bq) / sqrt(embed_dim), fp32 [C] (folded by the host binding; the
 * bk.q term is common to all encoders and cancels in the softmax). Outputs: out [B,T,C] bf16, weights [B,E] fp32.
 * partial_ws: merv_fusion_workspace_floats(B,E,T) floats.
 */
size_t merv_fusion_workspace_floats(int32_t batch, int32_t num_encoders, int32_t T);
int merv_fusion_forward(const void *const *v, int32_t num_encoders, int32_t batch, int32_t T, int32_t C,
                        const float *u, float *partial_ws, float *weights_out, void *out, void *stream);

/* Splice (merv/models/vidlms/merv.py:633-640): out[b] = cat(emb[b,:bos], vis[b], emb[b,bos:]) ; all bf16. */
int merv_splice_forward(const void *emb, const void *vis, int32_t batch, int32_t S, int32_t T, int32_t C,
                        int32_t bos, void *out, void *stream);

/*
 * ---- backward of the trainable tail ----
 * What torch autograd computes for the reference under loss.backward() (merv/training/strategies/base_strategy.py,
 * the `normalized_loss.backward()` of run_training) through CrossAttentionAdapterLearnableQuery.forward
 * (merv/util/nn_utils.py:487-521) and AveragePooling3DProjector.forward (nn_utils.py:320-330). The encoders are
 * frozen (merv.py:562), so no gradient flows past the pooled encoder tokens.
 *
 * Fusion: out = sum_e w_e V_e, w = softmax_e(mean_t(V_e) . u).
 *   merv_fusion_backward_reduce: dw[b,e] = sum_{t,c} grad_out[b,t,c] V_e[b,t,c] and vbar[b,e,:] = mean_t V_e (fp32).
 *     The binding then forms ds = w * (dw - sum_e w dw) and du = sum_{b,e} ds[b,e] vbar[b,e,:] (B x E scalars).
 *   merv_fusion_backward_mix:    dV_e = w_e grad_out + (ds_e / T) u, bf16, one tensor per encoder.
 * ws: merv_fusion_backward_workspace_floats(B,E,T,C) floats.
 */
size_t merv_fusion_backward_workspace_floats(int32_t batch, int32_t num_encoders, int32_t T, int32_t C);
int merv_fusion_backward_reduce(const void *const *v, int32_t num_encoders, int32_t batch, int32_t T, int32_t C,
                                const void *grad_out, float *ws, float *dw_out, float *vbar_out, void *stream);
int merv_fusion_backward_mix(const void *grad_out, const float *weights, const float *ds, const float *u,
                             int32_t num_encoders, int32_t batch, int32_t T, int32_t C, void *const *dv_out,
                             void *stream);

/*
 * Projector: Y = pooled W^T + b with pooled [M, C] (the `pooled_ws` buffer merv_projector_forward filled), Y [M, llm].
 *   grad_w [llm, C] bf16 = grad_out^T pooled  (two transposes + the forward GEMM kernel, fp32 accumulation over M)
 *   grad_b [llm] fp32    = column sums of grad_out
 * C % 128 == 0, llm % 8 == 0. ws: merv_projector_backward_workspace_bytes(M, C, llm) bytes, 256-byte aligned.
 */
size_t merv_projector_backward_workspace_bytes(int32_t M, int32_t C, int32_t llm_dim);
int merv_projector_backward(const void *grad_out, const void *pooled, int32_t M, int32_t C, int32_t llm_dim,
                            void *ws, size_t ws_bytes, void *grad_w, float *grad_b, void *stream);

/*
 * ---- LayerNorm folded into the GEMM that consumes it (bf16 path; the Python binding enables it by default) ----
 * For LN1 -> qkv and LN2 -> fc1 of every block
 *   Linear(LayerNorm(x)) = rstd * (x . (W*gamma)^T) - rstd * mean * colsum(W*gamma) + (W . beta + bias)
 * is exact algebra, so the encoder computes only the per-row statistics (one read of x instead of a read + write of the
 * normalised copy) and the GEMM reads the residual stream directly; its epilogue applies the row scale and the rank-1
 * correction in fp32. Rounding points differ from the reference's bf16(LayerNorm(x)): the weight product gamma*W is
 * rounded to bf16 once more, the activations are not rounded at all. The library writes the folded weights into `buf`
 * (merv_encoder_ln_fold_bytes(enc) bytes, 256-byte aligned, caller-owned). Ignored while MXFP8 mode is on. Call
 * merv_encoder_workspace_bytes AFTER enabling.
 */
size_t merv_encoder_ln_fold_bytes(const merv_encoder *enc);
int merv_encoder_enable_ln_fold(merv_encoder *enc, void *buf, size_t bytes, void *stream);

/*
 * ---- MXFP8 mode ("fp8 MFMA encoder GEMMs"); opt-in, never the default ----
 * OCP Microscaling FP8: e4m3 elements, one E8M0 scale per 32 consecutive k (shared exponent floor(log2 amax) - 8, plus
 * one when the scaled block maximum would exceed 448 so that nothing saturates; round-to-nearest-even), consumed by
 * v_mfma_scale_f32_16x16x128_f8f6f4 at twice the bf16 MFMA rate. There is no counterpart in the reference (it runs bf16
 * autocast, merv.py:816): this mode trades the bf16 tolerance for throughput.
 * Encoder in MXFP8 mode: the GEMMs of every block (qkv, attention out-projection, fc1, fc2, and LanguageBind's temporal
 * qkv / out-projection) run on MXFP8 operands; LayerNorm statistics, attention, the patch embedding and the residual
 * stream stay bf16 / fp32. The library quantises the block weights it was given at merv_encoder_create into `buf`
 * (merv_encoder_mxfp8_bytes(enc) bytes, 256-byte aligned, owned by the caller for the encoder's lifetime). Call
 * merv_encoder_workspace_bytes AFTER enabling: the workspace grows by the quantised activation buffer. dim and mlp_dim
 * must be multiples of 256 (>= 512).
 */
size_t merv_encoder_mxfp8_bytes(const merv_encoder *enc);
int merv_encoder_enable_mxfp8(merv_encoder *enc, void *buf, size_t bytes, void *stream);
/* Orchestration hint (round 6). When several encoders run concurrently, the chain that ENDS the step (the largest encoder's) should take the
 * fast, wide form for its sub-round GEMM launches (fewer than 72 tiles of 256 x 256: 136-150 small-tile blocks), while the chains that run beside
 * it keep the narrow one (39-68 eight-phase blocks from 32 tiles on) and cut their wide launches of up to a round (qkv, fc1) into consecutive
 * launches of at most 160 tiles, which leaves CUs to it: one video per step 9.43 -> 8.8-9.05 ms. `critical` != 0 (the default: a lone encoder is
 * its own critical chain) selects the first, 0 the second. Results are bit-identical either way (rows are independent). Mirrors nothing
 * in the reference (its encoders run one after the other, merv.py:563-566). */
int merv_encoder_set_latency_critical(merv_encoder *enc, int32_t critical);
/* Which block GEMMs run on MXFP8 once the mode is enabled: bit 0 qkv (and the temporal qkv), bit 1 attention
 * out-projection (and the temporal one), bit 2 fc1, bit 3 fc2; default 15. The others stay bf16 (accuracy / speed dial). */
int merv_encoder_set_mxfp8_mask(merv_encoder *enc, int32_t mask);

/* ---- single kernels, exported for parity tests and micro-benchmarks ---- */
/*
 * merv_quantize_mxfp8: x bf16 [rows, K] (ld elements) -> q [rows, K] bytes + scales (merv_mxfp8_scale_bytes(rows, K)
 *   bytes, in the GEMM's lane order: [K/128][ceil(rows/64)][(kblock%4)*16 + row%16][(row%64)/16]). K % 128 == 0.
 * merv_gemm_mxfp8: C[M,N] bf16 = epilogue(A8 . W8^T), same epilogue arguments as merv_gemm_bf16 (bias, activation,
 *   LayerScale, residual). K % 256 == 0, K >= 512, N % 256 == 0; lda / ldw in elements (= bytes), multiples of 16.
 */
size_t merv_mxfp8_scale_bytes(int32_t rows, int32_t K);
int merv_quantize_mxfp8(const void *x, int32_t rows, int32_t K, int32_t ld, void *q, void *scales, void *stream);
int merv_gemm_mxfp8(const void *A8, const void *scale_a, const void *W8, const void *scale_w, void *C, const float *bias,
                    const float *lscale, const void *res, int32_t M, int32_t N, int32_t K, int32_t lda, int32_t ldw,
                    int32_t ldc, int32_t ldres, int32_t act, void *stream);

/* out[c][r] = in[r][c] (bf16), columns R..Rpad-1 of `out` zero-filled; ldi, ldo, Rpad even. */
int merv_transpose_bf16(const void *in, int32_t R, int32_t C, int32_t ldi, void *out, int32_t ldo, int32_t Rpad,
                        void *stream);
int merv_gemm_bf16(const void *A, const void *W, void *C, const float *bias, const float *lscale, const void *res,
                   int32_t M, int32_t N, int32_t K, int32_t lda, int32_t ldw, int32_t ldc, int32_t ldres,
                   int32_t res_row_mod, int32_t out_group, int32_t out_stride, int32_t out_off, int32_t act,
                   void *stream);
int merv_layernorm(void *x, void *y, const float *gamma, const float *beta, const float *add, int32_t M, int32_t D,
                   int32_t add_div, int32_t add_mod, float eps, void *stream);
int merv_attention(const void *qkv, void *out, int32_t nseq, int32_t L, int32_t heads, int32_t D, float scale,
                   void *stream);
int merv_temporal_attention(const void *qkv, void *out, int32_t nclips, int32_t t, int32_t ntok, int32_t heads,
                            int32_t D, float scale, void *stream);
int merv_im2col(const void *pix, int32_t pix_dtype, void *out, int32_t B, int32_t frames, int32_t img, int32_t patch,
                int32_t tubelet, int32_t k_pad, int64_t sB, int64_t sF, int64_t sC, void *stream);
int merv_pool3d(const void *tokens, void *out, int32_t B, int32_t T, int32_t S, int32_t out_size, int32_t C,
                void *stream);

/*
 * Frame preprocessing on the GPU: uint8 frames [T,3,H,W] (device) -> normalised pixels.
 *  merv_preprocess_pil: torchvision Resize((S,S)) on a PIL image + ToTensor + Normalize, i.e. the DINOv2 / SigLIP
 *    (filter 1 = bicubic) and ViViT (filter 0 = bilinear) transforms (dinov2_video.py:76-124, siglip.py:86-134,
 *    vivit.py:50-92). The resized uint8 image is bit-exact with Pillow's Image.resize; out [T,3,S,S] fp32 or bf16;
 *    resized_u8 (optional, [T,3,S,S] uint8) exposes the intermediate for parity tests.
 *  merv_preprocess_languagebind: x/255 -> (x-mean)/std -> bilinear (align_corners=False) short side S -> centre crop S
 *    -> optional horizontal flip; out [3,T,S,S] (languagebind/video/processing_video.py:63-79; the reference flips at
 *    random, here `flip` is explicit).
 */
size_t merv_preprocess_workspace_bytes(int32_t T, int32_t H, int32_t W, int32_t out_size);
int merv_preprocess_pil(const void *frames_u8, int32_t T, int32_t H, int32_t W, int32_t out_size, int32_t filter,
                        const float *mean3, const float *std3, void *out_pixels, int32_t out_dtype, void *resized_u8,
                        void *workspace, size_t workspace_bytes, void *stream);
int merv_preprocess_languagebind(const void *frames_u8, int32_t T, int32_t H, int32_t W, int32_t out_size, int32_t flip,
                                 const float *mean3, const float *std3, void *out_pixels, int32_t out_dtype, void *stream);

/* 1 when this build of the library has its tuning hooks compiled in (-DMERV_TUNING_HOOKS: merv_amd/lib/libmerv_hip_hooks.so, the test /
 * probe build of the same sources), 0 for the product library: that one reads no environment variable and keeps no process-global
 * switch -- kernel selection is a function of a call's arguments alone -- and the two setters below are no-ops in it. */
int merv_tuning_hooks(void);
/* Tuning / test hook (hooks build only): force the GEMM tile configuration (low byte: 0 auto, 1: 128x128 two-deep ring, 3: 256x128,
 * 4: 256x128 with staggered half-blocks, 6: 128x128 four-deep ring, 7: 256x256 eight-phase where the shape allows it;
 * second byte: tile-order group size, 0 = default). */
void merv_debug_set_gemm_variant(int32_t variant);
/* Tuning / test hook (hooks build only): the attention kernels' deferred-max threshold in binary orders of magnitude (a lane's exponentials may sum to
 * 2^thr before its softmax reference moves); 0 = exact running maximum, default 8, values outside [0, 64] restore the default. */
void merv_debug_set_attn_rescale_thr(float thr);
/* Experiment hook (hooks build only; a no-op in the product): GEMM launches on `main_stream` put their remaining-rows launch on `aux_stream`
 * (event-forked before the main launch, event-joined behind it), so that it can start in its own main launch's tail. main_stream = NULL
 * clears every registration. Round 6: measured, not kept (profiles/r06_remainder_fork.json). */
void merv_debug_set_rest_fork(void *main_stream, void *aux_stream);
/* Test hook: plain bf16 GEMM (A [M,K], W [N,K]) whose epilogue writes its result as MXFP8 (q [M,N] + block scales). */
int merv_debug_gemm_mx_out(const void *A, const void *W, void *C_unused, int32_t M, int32_t N, int32_t K, void *q_out,
                           void *scales_out, void *stream);
/* Test hook: the MXFP8 GEMM with every epilogue term the encoder stacks use in MXFP8 mode under the LayerNorm fold (round 6) -- folded
 * LayerNorm (row_stats [M][2], ln_colsum [N]), LayerNorm partials out (stats_out [N/64][M][2]), LanguageBind's row-indexed add, an MXFP8
 * copy of the result beside bf16 C (keep_c = 1) or instead of it (keep_c = 0) -- and no_static_form = 1 keeps the run-time epilogue form,
 * so that the static (whole-tile) forms can be compared with it bit for bit. Contiguous operands (lda = ldw = K, ldc = ldres = N). */
int merv_debug_gemm_mxfp8_forms(const void *A8, const void *scale_a, const void *W8, const void *scale_w, void *C, const float *bias,
                                const float *lscale, const void *res, int32_t M, int32_t N, int32_t K, int32_t act,
                                const float *row_stats, const float *ln_colsum, float *stats_out, const float *row_add,
                                int32_t row_add_div, int32_t row_add_mod, void *mx_out_q, void *mx_out_scales, int32_t keep_c,
                                int32_t no_static_form, void *stream);
/* test hook: the bf16 GEMM with the LayerNorm-partials output the encoder requests from the GEMMs that write its residual
 * stream: per row, per 64 output columns, {sum, M2 about the 64-column mean} of the bf16-rounded values stored
 * ([N/64][M][2] floats: column tile major), which a one-thread-per-row kernel combines (Chan) into the statistics of a LayerNorm folded into
 * the next GEMM. */
int merv_debug_gemm_stats(const void *A, const void *W, void *C, const float *bias, const float *lscale, const void *res,
                          int32_t M, int32_t N, int32_t K, int32_t act, float *stats_out, void *stream);
/* test hook: C = bf16(bf16(A W^T + bias + res) + row_add[(m / row_add_div) % row_add_mod]) (row_add fp32 [row_add_mod, N]; the form
 * LanguageBind's fc2 uses to add the next block's temporal embedding) + the LayerNorm partials of the result */
int merv_debug_gemm_row_add(const void *A, const void *W, void *C, const float *bias, const void *res, int32_t M, int32_t N, int32_t K,
                            const float *row_add, int32_t row_add_div, int32_t row_add_mod, float *stats_out, void *stream);

/*
 * Per-launch HIP-event timing (bench.py roofline leg). While a class (bit of `class_mask`) is enabled every launch of it is
 * bracketed by two events on its own stream; merv_prof_read sums elapsed ms / launches / algorithmic FLOPs / algorithmic
 * bytes since the last reset.
 *   call level (a merv_gemm_bf16 call may be two kernel launches: eight-phase part + remaining rows):
 *     0 GEMM calls   1 attention calls   2 temporal attention   3 LayerNorm kernel
 *   kernel level (one bracket per kernel launch; together with 2 and 3 they partition the kernels of an encoder step):
 *     5 gemm_bf16_8phase_kernel without activation   6 gemm_bf16_8phase_kernel with an activation epilogue (fc1)
 *     7 gemm_bf16_kernel (rows the eight-phase launch left over, patch embedding, small problems)
 *     8 attn_kernel, K / V resident in LDS (257 / 261 tokens)   9 attn_kernel, K / V streamed (196 / 3137 tokens)
 *     10 row_stats + stats_finalize   11 pool + fusion score + fusion mix   12 im2col / prefix rows / token gather
 * Enable call-level and kernel-level classes in separate passes (nested brackets would time each other's event records).
 */
void merv_prof_enable(int32_t class_mask);
void merv_prof_reset(void);
int merv_prof_read(int32_t cls, double *total_ms, int64_t *launches, double *flops, double *bytes);

/*
 * Batch-1 token decode of the LLM hand-off: the per-token forward HF GenerationMixin runs for
 * the reference's generate() (merv/models/vidlms/merv.py:818-825 -> LlamaForCausalLM.forward with a KV cache). A decode step is
 * 5 launches per layer of these HBM-bound kernels instead of ~35 PyTorch ones; the prompt prefill keeps its GEMMs on the library
 * (PyTorch-ROCm) and takes the merv_prefill_* / merv_add_rmsnorm / merv_silu_mul calls below for everything between them.
 * bf16 tensors, fp32 accumulation, bf16 rounding wherever the module materialises a bf16 tensor.
 *  merv_decode_rmsnorm     LlamaRMSNorm: y = w * bf16(x * rsqrt(mean(x^2) + eps)); x, y [rows, D], w [D]
 *  merv_decode_gemv        nn.Linear at M = 1: y[N] = bf16(W[N,K] x[K]) (+ res[N]); with W2: y = silu(bf16(W x)) * bf16(W2 x)
 *                          (LlamaMLP's act_fn(gate_proj(x)) * up_proj(x)); y32 != NULL: fp32 output instead (logits);
 *                          norm_w != NULL: the RMSNorm of the input fused in (x is the raw residual stream; bit-identical to
 *                          merv_decode_rmsnorm followed by the plain call; K <= 16384)
 *  merv_decode_rope_cache  apply_rotary_pos_emb at position *pos (device int64) on q [H*hd] -> q_out and k [Hkv*hd] -> k_cache[:, *pos],
 *                          v -> v_cache[:, *pos]; caches [Hkv, max_len, hd], cos / sin tables [max_len, hd] bf16
 *  merv_decode_attention   out[H*hd] = softmax(q K^T * scale) V over cache positions 0..*pos (GQA: kv head = h / (H/Hkv)),
 *                          split over `nsplit` position ranges; ws: merv_decode_attention_workspace_floats(H, nsplit) floats. hd = 128.
 * The position comes from device memory so that a step captured in a hipGraph replays at every position.
 */
int merv_decode_rmsnorm(const void *x, const void *w, void *y, int32_t rows, int32_t D, float eps, void *stream);
int merv_decode_gemv(const void *W, const void *W2, const void *x, const void *res, void *y, float *y32, int32_t N, int32_t K,
                     const void *norm_w, float norm_eps, void *stream);
int merv_decode_rope_cache(const void *q, const void *k, const void *v, void *q_out, void *k_cache, void *v_cache,
                           const void *cos_t, const void *sin_t, const int64_t *pos, int32_t H, int32_t Hkv, int32_t hd,
                           int32_t max_len, void *stream);
/* Prompt prefill (batch 1; S positions at once) -- the elementwise parts of a decoder layer between the library GEMMs, each one launch
 * instead of the 5-10 PyTorch kernels of the module's expression (same rounding points; merv/models/vidlms/merv.py:723-734 ->
 * LlamaDecoderLayer.forward): merv_decode_rmsnorm takes rows = S; these two do the rest.
 *  merv_prefill_rope_cache  apply_rotary_pos_emb on positions pos0 .. pos0 + S - 1: q [S, ldq] (H*hd columns) rotated IN PLACE,
 *                           rot(k [S, ldk]) -> k_cache[:, pos0 + s], v [S, ldk] -> v_cache[:, pos0 + s] (q / k / v may be column ranges of
 *                           one projection output); caches [Hkv, max_len, hd], tables [max_len, hd]; hd % 16 == 0
 *  merv_silu_mul            out = bf16(bf16(silu(gate)) * up), n elements (n % 8 == 0); out may alias gate or up
 *  merv_add_rmsnorm         the residual add and the next RMSNorm in one pass: x <- bf16(x + delta) IN PLACE, y = RMSNorm(x) (same bits
 *                           as the add followed by merv_decode_rmsnorm); x, delta, y [rows, D], D <= 8192
 *  merv_prefill_attention   causal softmax(q k^T * scale) v of ONE sequence of S positions, hd = 128, GQA (kv head = h / (H / Hkv)):
 *                           replaces F.scaled_dot_product_attention(q, k, v, is_causal=True) of LlamaAttention.forward on the prompt.
 *                           q [S, ldq] (head h at columns 128 h ..; rotary applied), k / v: kv head g, position s at
 *                           base + g * kv_head_stride + s * ldk (the KV cache itself: ldk = 128, kv_head_stride = max_len * 128),
 *                           out [S, ldo] in q's column layout -- the o-projection's input, no transpose */
int merv_prefill_rope_cache(void *q, const void *k, const void *v, void *k_cache, void *v_cache, const void *cos_t, const void *sin_t,
                            int32_t S, int32_t pos0, int32_t H, int32_t Hkv, int32_t hd, int32_t max_len, int32_t ldq, int32_t ldk,
                            void *stream);
int merv_silu_mul(const void *gate, const void *up, void *out, int64_t n, void *stream);
int merv_add_rmsnorm(void *x, const void *delta, const void *w, void *y, int32_t rows, int32_t D, float eps, void *stream);
int merv_prefill_attention(const void *q, const void *k, const void *v, void *out, int32_t S, int32_t H, int32_t Hkv, int32_t hd,
                           int32_t ldq, int32_t ldk, int64_t kv_head_stride, int32_t ldo, float scale, void *stream);
/* three projections of the same input in one launch (q_proj / k_proj / v_proj): y_i[N_i] = bf16(W_i[N_i,K] x[K]) */
int merv_decode_gemv3(const void *Wa, const void *Wb, const void *Wc, const void *x, void *ya, void *yb, void *yc,
                      int32_t Na, int32_t Nb, int32_t Nc, int32_t K, const void *norm_w, float norm_eps, void *stream);
/* the same with nn.Linear biases (bf16 [N_i] or NULL each): Qwen2's q / k / v projections */
int merv_decode_gemv3_bias(const void *Wa, const void *Wb, const void *Wc, const void *x, void *ya, void *yb, void *yc,
                           int32_t Na, int32_t Nb, int32_t Nc, int32_t K, const void *norm_w, float norm_eps,
                           const void *bias_a, const void *bias_b, const void *bias_c, void *stream);
size_t merv_decode_attention_workspace_floats(int32_t H, int32_t nsplit);
int merv_decode_attention(const void *q, const void *k_cache, const void *v_cache, void *out, float *ws, const int64_t *pos,
                          int32_t H, int32_t Hkv, int32_t hd, int32_t max_len, int32_t nsplit, float scale, void *stream);
/* merv_decode_rope_cache + merv_decode_attention as ONE launch (bit-identical result): every block rotates its head's query, the
 * token being decoded is rotated from the raw k / v and used from registers (cache[*pos] is written for later steps, never
 * read here), and the block that arrives last on its head's counter merges the splits. ws: ..._fused_workspace_floats(H, nsplit)
 * floats, ZEROED by the caller once (the counters at its end return to zero after every launch). */
size_t merv_decode_attention_fused_workspace_floats(int32_t H, int32_t nsplit);
int merv_decode_attention_fused(const void *q, const void *k, const void *v, const void *cos_t, const void *sin_t, const int64_t *pos,
                                void *k_cache, void *v_cache, void *out, float *ws, int32_t H, int32_t Hkv, int32_t hd,
                                int32_t max_len, int32_t nsplit, float scale, void *stream);
/* merv_decode_attention_split with a read-only pass over the NEXT launch's weights riding on it (round 6): the split attention is a chain of
 * dependent round trips over ~17 MB of cache that leaves HBM idle for its ~7 us; `next_w_bytes / next_block_bytes` extra workgroups behind the
 * H x nsplit attention ones each read `next_block_bytes` of `next_w` -- for the o-projection that follows: W_o, in slices of the 16 rows one
 * workgroup of merv_decode_oproj_merge reads -- and, workgroups going to the 8 XCDs round-robin (H * nsplit % 8 == 0 required), prefetch workgroup
 * b lands on the XCD whose L2 workgroup b of the next launch reads through. Same results as merv_decode_attention_split (next_w = NULL: the same
 * launch). Replaces nothing in the reference: it is how the five launches per layer of HF's LlamaDecoderLayer.forward overlap here. */
int merv_decode_attention_split_prefetch(const void *q, const void *k, const void *v, const void *cos_t, const void *sin_t,
                                         const int64_t *pos, void *k_cache, void *v_cache, float *ws, int32_t H, int32_t Hkv, int32_t hd,
                                         int32_t max_len, int32_t nsplit, float scale, const void *next_w, int64_t next_w_bytes,
                                         int32_t next_block_bytes, void *stream);
/* The same two steps with the merge moved into the o-projection (round 4; bit-identical to merv_decode_attention_fused followed by
 * merv_decode_gemv(Wo, NULL, out, x, x, ...)): merv_decode_attention_split ends at the split partials (ws:
 * merv_decode_attention_split_workspace_floats(H, nsplit) floats, 16-byte aligned, records of 132; no counters, no `out`, nothing to
 * zero), merv_decode_oproj_merge computes
 * y[N] = res[N] + Wo[N, H*hd] . merge(ws), merging while its first weight loads are in flight, and optionally stores the merged
 * attention output [H*hd] (attn_out, NULL to skip). 9.0 + 9.3 us per layer against 13.8 + 9.3 at 1050 positions. */
size_t merv_decode_attention_split_workspace_floats(int32_t H, int32_t nsplit);
int merv_decode_attention_split(const void *q, const void *k, const void *v, const void *cos_t, const void *sin_t, const int64_t *pos,
                                void *k_cache, void *v_cache, float *ws, int32_t H, int32_t Hkv, int32_t hd, int32_t max_len,
                                int32_t nsplit, float scale, void *stream);
int merv_decode_oproj_merge(const void *Wo, const void *res, void *y, const float *ws, void *attn_out, int32_t N, int32_t H, int32_t hd,
                            int32_t nsplit, void *stream);
/* Greedy decoding inside a captured step (HF GenerationMixin's greedy search: next token = argmax of the last logits,
 * merv/models/vidlms/merv.py:818-825 with do_sample=False): tok[0] <- argmax(logits[V]) by torch.argmax's rule (the first maximum; a NaN
 * wins), out_tokens[*pos - pos0] <- the token (out_tokens may be NULL), *pos += 1 -- so that a replayed step leaves the next step's
 * token and position on the device and the host loop launches nothing else per token. */
int merv_decode_greedy_advance(const float *logits, int32_t V, int64_t *tok, int64_t *pos, int64_t *out_tokens, int64_t pos0, void *stream);
/* The same hand-over with the token DRAWN from softmax(logits / temperature) -- `do_sample=True, temperature=T` of the reference's
 * generate() kwargs (scripts/quick_start.py:24-32 -> merv.py:818-825 -> HF GenerationMixin's sampling step: logits / T, softmax,
 * torch.multinomial) -- as argmax_i(logits_i / T + Gumbel_i): the Gumbel-max trick draws from exactly that categorical distribution
 * in one pass. The Gumbel variates come from Philox4x32-10 keyed by `seed` with counter (i / 4, *pos), so a captured step replays with
 * fresh numbers at every position and (seed, position) is reproducible. `params` is a 32-byte block in DEVICE memory, 8-byte aligned,
 * read by the kernel (nothing of it is baked into a captured graph):
 *   float inv_temperature; int32 eos_id (< 0: none); uint64 seed; int64 min_new_tokens; int64 first_pos -- eos_id cannot be drawn
 *   as new token number < min_new_tokens, where the step at position first_pos draws token number 1 (HF
 *   MinNewTokensLengthLogitsProcessor; number 0 is the token drawn from the prompt's logits).
 * top-k / top-p / repetition penalty are not implemented here (merv_amd/llm.py keeps them on its host loop). */
int merv_decode_sample_advance(const float *logits, int32_t V, const void *params, int64_t *tok, int64_t *pos, int64_t *out_tokens,
                               int64_t pos0, void *stream);
/* The attention step of timm's AttentionPoolLatent (global_pool='map': what the SigLIP ids without `all-no-cls` return,
 * siglip.py:46-63): one learnt query per head against every token of a frame. kv [nseq*ntok, 2*D] bf16 = [k | v] rows (the kv
 * Linear's output), q [D] fp32 = q Linear of the latent, out [nseq, D] bf16; D = heads * 64, ntok <= 1024. */
int merv_map_pool_attention(const void *kv, const float *q, void *out, int32_t nseq, int32_t ntok, int32_t heads, float scale,
                            void *stream);

/*
 * A paged key / value cache for batches of rows (sequences) of unlike length, and the attention of one new token for each row over it. The
 * reference decodes through HF's DynamicCache, one clip a call (merv/models/vidlms/merv.py:818-825); these carry the decoding step of several clips
 * or questions at once (merv_amd/paged.py, PagedDecoder). They came after ABI version 4's other entries and change none of them.
 *
 *  Pages: k_pages / v_pages hold element (page, kv head, slot, d) at page * stride_page + head * stride_head + slot * stride_token + d (the same strides
 *  for both), bf16 or OCP e4m3. With e4m3, scale byte (page, head, slot) is at page * scale_stride_page + head * scale_stride_head + slot and a number
 *  stands for code * 2^(byte - 127). table[row * table_stride + i] is the page that holds positions i * page_size .. of a row; entries no call reaches
 *  may hold anything. Device-side integers are never trusted with an address: see each call for what a bad one does.
 *  Limits: head_dim 64 or 128; page_size a power of two from 16 to 1024; page and row pointers 16-byte aligned with strides that are multiples of 8 (bf16) or 16
 *  (e4m3) elements, scale pointers 4-byte aligned with strides that are multiples of 4. A write takes up to 2^28 vectors (keys, values and queries), a
 *  read 2^27 keys, an attention under 2^22 rows x heads, 2^30 positions a row and under 2^31 units of 128 positions over all rows and heads.
 */
enum { MERV_KV_BF16 = 0, MERV_KV_E4M3 = 1 };
typedef struct merv_paged_cache {
    void *k_pages, *v_pages;
    void *k_scales, *v_scales;    /* e4m3 only, else NULL */
    const int32_t *table;         /* device [rows, table_width] */
    int64_t n_pages;
    int64_t stride_page, stride_head, stride_token;      /* in elements */
    int64_t scale_stride_page, scale_stride_head;
    int64_t table_stride;
    int32_t rows, table_width, kv_heads, head_dim, page_size, format;
} merv_paged_cache;
/* New tokens into the cache: apply_rotary_pos_emb on k (and q), then the store; v as it is. Token t (0 <= t < T) is row b's where
 * offsets[b] <= t < offsets[b + 1] (device int32 [rows + 1], not decreasing), at position start[b] + t - offsets[b]; offsets = NULL: one token
 * a row, T = rows. A row with start[b] < 0 and tokens at or behind offsets[rows] are left alone in every output. k, v [T, kv_heads, hd], q, q_out
 * [T, heads, hd], k_out [T, kv_heads, hd] bf16 with token and head strides in elements; q = NULL (heads = 0) and k_out = NULL leave these out; q_out may be q
 * and k_out may be k, of the same strides; they share no memory with any other operand (two that begin at the same address are refused).
 * cos, sin [rope_len, hd] bf16, row stride rope_stride; both NULL: no rotation (q must be NULL). rot = x cos + rotate_half(x) sin in fp32,
 * rounded to bf16 once. e4m3: a row's scale is the smallest power of two under which no finite element of the (bf16) row is over 448, 2^-126 at least;
 * the codes are rounded to nearest even (248 x 2^120 and more to 2^128, which reads back as infinity); NaN and infinities become NaN.
 * A position without a page in the table is not stored; with rotation, one
 * outside the tables or without a page is NaN in q_out and k_out. Two tokens of one call must not meet in one slot of one page. */
int merv_paged_cache_write(const merv_paged_cache *cache, const void *k, int64_t k_stride, int64_t k_head_stride, const void *v, int64_t v_stride,
                           int64_t v_head_stride, const void *q, int64_t q_stride, int64_t q_head_stride, const void *cos_t, const void *sin_t,
                           int64_t rope_len, int64_t rope_stride, void *q_out, int64_t q_out_stride, int64_t q_out_head_stride, void *k_out,
                           int64_t k_out_stride, int64_t k_out_head_stride, const int32_t *offsets, const int32_t *start, int32_t T, int32_t heads,
                           void *stream);
/* Cached keys and values back as bf16: k_out, v_out [T, kv_heads, hd]; token t is row b's (offsets as above, required) at position
 * (start ? start[b] : 0) + t - offsets[b]. A position without a page reads as NaN; rows with start[b] < 0 and tokens behind the last row are left alone.
 * k_out and v_out share no memory with each other or the cache. */
int merv_paged_cache_read(const merv_paged_cache *cache, void *k_out, int64_t k_out_stride, int64_t k_out_head_stride, void *v_out, int64_t v_out_stride,
                          int64_t v_out_head_stride, const int32_t *offsets, const int32_t *start, int32_t T, void *stream);
/* out[b, h] = sum_j softmax_j(scale * q[b, h] . k[b, j]) v[b, j] over positions max(0, len - window) .. len - 1 of row b, len = lens[b] (device int32;
 * window <= 0: all); kv head = h / (heads / kv_heads). lse (may be NULL) [rows, heads] fp32 = ln sum_j exp(scale * q . k). len <= 0: out = 0 and lse = -inf. A
 * length over the table's capacity or a bad page among those the row reads: that row's out and lse are NaN. Keys and values behind a row's length,
 * in its last page or before its window, may hold anything, NaN among it. q, out [rows, heads, hd] bf16 by strides (out may be q, of the same strides); workspace:
 * merv_paged_decode_attention_workspace_bytes(...) bytes, 16-byte aligned, of any contents, not shared by calls that may run at the same time. */
size_t merv_paged_decode_attention_workspace_bytes(int32_t rows, int32_t heads, int32_t kv_heads, int32_t head_dim, int64_t capacity);
int merv_paged_decode_attention(const merv_paged_cache *cache, const void *q, int64_t q_stride, int64_t q_head_stride, void *out, int64_t out_stride,
                                int64_t out_head_stride, float *lse, const int32_t *lens, int32_t heads, int64_t window, float scale, void *workspace,
                                size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* MERV_HIP_H */
