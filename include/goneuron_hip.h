/*
 * goneuron_hip.h — C ABI of libgoneuron_hip.so, the MI355X (gfx950) training
 * backend for GoNeuron's fp32 training step (forward + backward + Adam).
 *
 * The library replaces the reference's per-sample CPU loop and its Metal cgo
 * bridge.  Every entry point below names the reference interface it stands in
 * for (paths relative to the GoNeuron tree).  Conventions:
 *   - every call returns an int status: GN_OK (0) or a negative GN_ERR_* code;
 *     gn_last_error() gives the message of the last failure on a context
 *     (the reference's Metal ABI returns void and drops errors,
 *     internal/layer/metal.go:270-274);
 *   - host pointers are read or written only during the call, never retained;
 *   - "_device" entry points take device pointers (HBM-resident inputs);
 *   - one HIP stream per context; a context is not thread-safe (the Go side
 *     serialises calls with a mutex, as MetalDevice.mu does, metal.go:70).
 */
#ifndef GONEURON_HIP_H
#define GONEURON_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes ------------------------------------------------------ */
#define GN_OK 0
#define GN_ERR_INVALID (-1)     /* bad argument (null, size, kind) */
#define GN_ERR_HIP (-2)         /* HIP runtime error */
#define GN_ERR_OOM (-3)         /* device allocation failed */
#define GN_ERR_UNSUPPORTED (-4) /* layer/activation combination not built */
#define GN_ERR_SHAPE (-5)       /* input size mismatch (layer.go:347-349) */
#define GN_ERR_INJECTED (-6)    /* forced by gn_debug_fail_next */
#define GN_ERR_NO_DEVICE (-7)   /* no HIP device */
#define GN_ERR_INDEX (-8)       /* index out of range (embedding.go:126-128) */

/* ---- activation codes ---------------------------------------------------
 * A layer carries the activation *object* the Go code was given and whether it
 * was a pointer (&activations.Softmax{}) or a value (activations.Softmax{}),
 * because Dense dispatches on cacheActivationType (layer.go:183-205), which
 * only recognises pointer Softmax/LogSoftmax: the facade's values run as
 * identity forward and NaN derivative (activations.go:150-158). */
#define GN_ACT_NIL 0
#define GN_ACT_RELU 1
#define GN_ACT_SIGMOID 2
#define GN_ACT_TANH 3
#define GN_ACT_SOFTMAX 4
#define GN_ACT_LOGSOFTMAX 5
#define GN_ACT_LINEAR 6
#define GN_ACT_GELU 7   /* value activations.GELU{}: identity forward, GELU' backward */

/* ---- layer kinds (the []layer.Layer given to goneuron.NewSequential) ----- */
#define GN_LAYER_DENSE 1         /* layer.NewDense            layer.go:267 */
#define GN_LAYER_DROPOUT 2       /* layer.NewDropout          dropout.go:47 */
#define GN_LAYER_CONV2D 3        /* layer.NewConv2D           conv2d.go:74 */
#define GN_LAYER_MAXPOOL2D 4     /* layer.NewMaxPool2D        maxpool2d.go:45 */
#define GN_LAYER_FLATTEN 5       /* layer.NewFlatten          reshape.go:29 */
#define GN_LAYER_EMBEDDING 6     /* layer.NewEmbedding        embedding.go */
#define GN_LAYER_POSENC 7        /* layer.NewPositionalEncoding transformer.go:51 */
#define GN_LAYER_TRANSFORMER 8   /* layer.NewTransformerBlockE transformer.go:908 */
#define GN_LAYER_CLSPOOL 9       /* layer.NewCLSPooling       transformer.go:1679 */
#define GN_LAYER_LSTM_UNROLLER 10 /* SequenceUnroller(LSTM)   unroller.go:57, lstm.go */
#define GN_LAYER_AVGPOOL2D 11    /* layer.NewAvgPool2D        avgpool2d.go:50 */
#define GN_LAYER_RMSNORM 12      /* layer.NewRMSNorm          rmsnorm.go:49 */
#define GN_LAYER_SWIGLU 13       /* layer.NewSwiGLU           swiglu.go:47 */
#define GN_LAYER_BATCHNORM2D 14  /* layer.NewBatchNorm2D      batchnorm2d.go:70 */
#define GN_LAYER_GRU_UNROLLER 15 /* SequenceUnroller(GRU)     unroller.go:57, gru.go:83 */
#define GN_LAYER_MOE 16          /* layer.NewMoE              moe.go:47 */
#define GN_LAYER_MHA 17          /* layer.NewMultiHeadAttentionE transformer.go:283 (dim, num_heads,
                                    seq_len, causal; parameters start at 0, transformer.go:367-379) */
#define GN_LAYER_LAYERNORM 18    /* layer.NewLayerNorm        layernorm.go:57 (dim = normalizedShape,
                                    eps; gamma 1, beta 0) */
#define GN_LAYER_GAP1D 19        /* layer.NewGlobalAveragePooling1D transformer.go:1524 (seq_len, dim) */

/* TransformerBlockExt options (layer.ActivationType, layer.NormType) */
#define GN_BLOCK_ACT_RELU 0
#define GN_BLOCK_ACT_SWIGLU 1
#define GN_BLOCK_ACT_GELU 2
#define GN_BLOCK_NORM_LN 0
#define GN_BLOCK_NORM_RMS 1

#define GN_LOSS_MSE 1            /* loss.MSE          loss.go:38-105 */
#define GN_LOSS_CE 2             /* loss.CrossEntropy loss.go:108-178 */

typedef struct gn_layer_desc {
  int32_t kind;
  int32_t in_size;      /* Dense in / Dropout & Flatten size / first-layer input length */
  int32_t out_size;     /* Dense out / LSTM hidden */
  int32_t act;          /* GN_ACT_* */
  int32_t act_is_ptr;   /* 1 when the Go activation is a pointer */
  int32_t in_channels;  /* Conv2D / MaxPool2D; -1 = lazy (MaxPool runs as 1 channel) */
  int32_t out_channels;
  int32_t kernel, stride, padding;
  float p;              /* Dropout probability */
  int32_t seq_len, num_heads, ff_dim, causal, vocab, dim; /* RMSNorm: dim = normalizedShape */
  int32_t return_sequences;
  float eps;            /* RMSNorm / LayerNorm eps; 0 selects the facade's 1e-5 (goneuron.go:220-236) */
  int32_t block_act;    /* TransformerBlock ff1: GN_BLOCK_ACT_* (transformer.go:199-203) */
  int32_t block_norm;   /* TransformerBlock norms: GN_BLOCK_NORM_* (transformer.go:205-210) */
  int32_t use_rope;     /* TransformerBlock: rotary embeddings on Q and K (transformer.go:212-236) */
  float momentum;       /* BatchNorm2D running-stat momentum, as given (the facade passes 0.1) */
  int32_t no_affine;    /* BatchNorm2D without gamma / beta (NewBatchNorm2D affine = false) */
  int32_t num_experts;  /* MoE experts (<= 64) */
  int32_t top_k;        /* MoE experts per sample */
} gn_layer_desc;

typedef struct gn_adam_desc {   /* opt.NewAdam opt.go:117-126 */
  float lr, beta1, beta2, eps;  /* zeros select the reference defaults */
} gn_adam_desc;

typedef struct gn_info {
  char arch[64];
  int32_t cu_count;
  int64_t hbm_bytes;
  double peak_fp32_mfma_tflops; /* dense fp32 matrix peak */
  double peak_hbm_gbps;
} gn_info;

typedef struct gn_ctx gn_ctx;
typedef struct gn_model gn_model;

/* ---- context -------------------------------------------------------------
 * Replaces layer.GetDefaultDevice / MetalDevice construction
 * (internal/layer/device.go:39-48, metal.go:76-98). */
int gn_available(void);                      /* 1 when a HIP device is present */
int gn_init(int device_ordinal, gn_ctx **out);
void gn_shutdown(gn_ctx *ctx);
const char *gn_last_error(const gn_ctx *ctx);
int gn_device_info(gn_ctx *ctx, gn_info *info);
int gn_sync(gn_ctx *ctx);                    /* waitForMetal, metal_ops.m:1002-1007 */
/* Test hook: the next entry point that takes this context fails with `code`. */
int gn_debug_fail_next(gn_ctx *ctx, int code);

/* ---- device buffers (createMetalBuffer / update / read, metal.go:6-50) --- */
int gn_malloc(gn_ctx *ctx, size_t bytes, void **dptr);
int gn_free(gn_ctx *ctx, void *dptr);
int gn_memcpy_h2d(gn_ctx *ctx, void *dst, const void *src, size_t bytes);
int gn_memcpy_d2h(gn_ctx *ctx, void *dst, const void *src, size_t bytes);
int gn_memset_zero(gn_ctx *ctx, void *dst, size_t bytes);

/* ---- model: Sequential.Compile + Network.initBuffers --------------------
 * sequential.go:26-87, net.go:91-127: layers are built with the reference's
 * seeded LCG initialisation into one device-resident flat arena
 * (params | grads | Adam m | Adam v).  `workers` is the trainBatchParallel
 * worker count W (net.go:588-608; 1 = trainBatchSequential). */
int gn_model_create(gn_ctx *ctx, const gn_layer_desc *layers, int32_t nlayers,
                    int32_t loss_kind, const gn_adam_desc *adam, int32_t max_batch,
                    int32_t workers, gn_model **out);
void gn_model_destroy(gn_model *m);
int gn_model_nparams(gn_model *m, int64_t *n);
int gn_model_layer_params(gn_model *m, int32_t layer, int64_t *offset, int64_t *count);
int gn_model_out_size(gn_model *m, int32_t *n);
/* The layers as built (a loaded model's descriptions) and the loss. */
int gn_model_layer_count(gn_model *m, int32_t *n);
int gn_model_layer_desc(gn_model *m, int32_t layer, gn_layer_desc *out);
int gn_model_loss_kind(gn_model *m, int32_t *loss_kind);
/* Network.Params / SetParams / Gradients (net.go:549-572, 787-846). */
int gn_model_get_params(gn_model *m, float *dst, int64_t offset, int64_t n);
int gn_model_set_params(gn_model *m, const float *src, int64_t offset, int64_t n);
int gn_model_get_grads(gn_model *m, float *dst, int64_t offset, int64_t n);
int gn_model_get_adam(gn_model *m, float *m_dst, float *v_dst, int64_t offset, int64_t n,
                      int32_t *timestep);
/* Restores Adam moments and the timestep (resume; the reference's
 * Adam.NewStep / StepInPlace state, opt.go:237-335). */
int gn_model_set_adam(gn_model *m, const float *m_src, const float *v_src, int64_t offset, int64_t n,
                      int32_t timestep);
/* Device pointers of the arena regions (for zero-copy callers). */
int gn_model_arena(gn_model *m, float **params, float **grads, float **adam_m, float **adam_v);

/* Network.TrainBatch (net.go:412-436): one fwd+bwd over B samples, gradient
 * average, Adam step.  Host inputs: x is B x in_size, y is B x out_size
 * (row major, the [][]float32 batches flattened).  loss_out may be NULL.
 * On failure: a step that failed before any parameter was updated leaves
 * the model as it was.  Large models update each layer as soon as its
 * backward is done; a step of such a model that fails after some layers
 * were updated leaves those at step t and the others at t-1 (reload a
 * checkpoint), with the Adam timestep at t, so a retry never applies bias
 * correction t twice. */
int gn_model_train_step(gn_model *m, const float *x, const float *y, int32_t B, float *loss_out);
/* Same with HBM-resident x / y; the mean loss stays on the device (read it
 * with gn_model_read_loss).  No host synchronisation. */
int gn_model_train_step_device(gn_model *m, const float *x_dev, const float *y_dev, int32_t B);
/* No counterpart in the reference (launch-overhead control).  Training steps
 * of models without MoE or LSTM layers replay their forward + loss + backward
 * launches from a HIP graph: the first step for a given (x, y, B, training
 * flags) runs eagerly, the second is captured, later ones replay it; Adam is
 * launched after it as usual.  Same kernels, same results.  on = 0 turns it
 * off (and frees the graphs), 1 back on (the default).  A model keeps at most
 * 4 graphs; gn_model_reserve frees them.  A replay reads x and y at the
 * addresses of the step it was captured from, which are the addresses its
 * key matched. */
int gn_model_set_graphs(gn_model *m, int32_t on);
/* Number of captured step graphs the model holds. */
int gn_model_graph_count(gn_model *m, int32_t *n);
/* Test hook (no counterpart in the reference): polls per wait of the
 * cooperative LSTM BPTT kernel before it reports a timeout (default 2^18);
 * a negative value makes every wait time out at once, so the error path
 * (GN_ERR_HIP at the next gn_model_read_loss / gn_model_train_step) can be
 * tested without a fault. */
int gn_debug_lstm_spin_limit(gn_model *model, int32_t polls);
/* Test hook (no counterpart in the reference): polls of the LSTM clip
 * kernel's wait for the Gram kernel it runs beside (default 2048).  When the
 * two kernels do not run at the same time (a profiler, a busy device) the
 * clip gives up after that many polls and a launch queued after the Gram
 * kernel clips the chain instead; 0 forces that path, whose results equal
 * the overlapped path's bit for bit. */
int gn_debug_lstm_clip_bail(gn_model *model, int32_t polls);
/* Test hook (no counterpart in the reference): on = 0 makes training passes
 * run the output Dense layer through its GEMMs, loss-row and column-sum
 * kernels even where it qualifies for the two fused output-layer kernels
 * (at most 32 outputs, input width a multiple of 4); 1 (the default) allows
 * them.  Both paths compute the same step to float32 rounding. */
int gn_debug_fused_tail(gn_model *model, int32_t on);
/* Test hook (no counterpart in the reference): on = 0 makes train steps of
 * small models (under 8 Mi parameters) run Network.Step's Adam update as a
 * launch of its own after the backward; 1 (the default) lets the backward's
 * last launch carry it where that launch writes the step's last gradients
 * (a first Conv2D's weight-gradient reduction).  Both give the same step bit
 * for bit. */
int gn_debug_step_update(gn_model *model, int32_t on);
/* Test hook (no counterpart in the reference): on = 1 runs the backward's
 * parameter-gradient kernels (Dense dW and bias sums, the transformer
 * block's token sums and weight gradients) on a second stream beside the
 * input-gradient kernels, as steps with per-layer Adam updates (models of
 * at least 8 Mi parameters) always do; 0 (the default) keeps them on the
 * main stream otherwise.  Both give the same step bit for bit. */
int gn_debug_side_streams(gn_model *model, int32_t on);
/* Forward + backward + average only (grads valid, no Adam step). */
int gn_model_accumulate_device(gn_model *m, const float *x_dev, const float *y_dev, int32_t B);
/* Network.Step (net.go:260-284): Adam.NewStep + StepInPlace on the arena. */
int gn_model_step(gn_model *m);
int gn_model_read_loss(gn_model *m, float *loss);
/* Sequential.Predict / PredictBatch (sequential.go:118-160): inference mode
 * forward of B samples; out is B x out_size. */
int gn_model_predict(gn_model *m, const float *x, int32_t B, float *out);
/* The same with HBM-resident x (B x in_size) and output (B x out_size); no
 * host synchronisation (the device-side ForwardBatch of sequential.go:145-160). */
int gn_model_predict_device(gn_model *m, const float *x_dev, int32_t B, float *out_dev);
/* gn_model_predict and a draw from each sample's outputs as logits, with
 * gn_sample's settings as host arrays of B (each but u may be NULL); ids: B
 * indices.  No counterpart in the reference.  The last layer must give logits or
 * log-probabilities: a Dense Softmax pointer is GN_ERR_UNSUPPORTED.  The draw is from
 * what the model puts out: behind a CLSPooling that is the pooled position, a next
 * token only if the model was trained to put one out there. */
int gn_model_sample(gn_model *m, const float *x, int32_t B, const float *temperature, const int32_t *top_k,
                    const float *top_p, const float *min_p, const float *u, int32_t *ids);
/* Network.SetTraining (net.go:187-193): sets the flag of every layer.  Layers
 * start as the reference constructs them (Dropout and BatchNorm2D in training
 * mode, MoE not: dropout.go:56, batchnorm2d.go:88, moe.go:46-90); Predict
 * turns the flags off and leaves them off (sequential.go:118-134).  With
 * workers > 1 a training step uses the flags of trainBatchParallel's worker
 * clones, which copy the network's flags when first needed and keep them
 * (net.go:129-152). */
int gn_model_set_training(gn_model *m, int32_t training);
int gn_model_get_training(gn_model *m, int32_t layer, int32_t *training);
/* Network.TrainBatch / PredictBatch accept any batch size (net.go:412-436):
 * grows the batch-sized buffers to max_batch samples, keeping parameters,
 * gradients, Adam state, running statistics, noise streams and flags.  A
 * smaller value is a no-op.  On failure the model keeps its old size. */
int gn_model_reserve(gn_model *m, int32_t max_batch);
/* Samples the last training step skipped because an Embedding index was out
 * of range: the reference's batch loop drops such a sample (net.go:738-741;
 * a trainBatchParallel worker drops the rest of its chunk and the chunk's
 * loss, net.go:641-655) and the step still applies.  Inference passes report
 * the same condition as GN_ERR_INDEX (ForwardBatch returns the error,
 * net.go:447-450). */
int gn_model_skipped_samples(gn_model *m, int32_t *count);
/* Layer probes for parity tests: saved output of `layer` for the last batch
 * (B x out_len); int32 indices of the last batch: MaxPool2D argmax switches
 * (B x out_len) or the MoE routes (B x k expert ids, routing order). */
int gn_model_layer_output(gn_model *m, int32_t layer, float *dst, int64_t n);
int gn_model_layer_argmax(gn_model *m, int32_t layer, int32_t *dst, int64_t n);
/* BatchNorm2D running statistics (C floats each) of `layer`:
 * GetRunningMean / GetRunningVar (batchnorm2d.go:837-838) and, for restoring
 * a checkpoint, writing them back (NamedParams running_mean / running_var,
 * batchnorm2d.go:755-767). */
int gn_model_get_running_stats(gn_model *m, int32_t layer, float *mean, float *var, int32_t n);
int gn_model_set_running_stats(gn_model *m, int32_t layer, const float *mean, const float *var,
                               int32_t n);

/* ---- checkpoints: the formats either side of training ------------------
 * Network.SaveBinaryWeights (net.go:1119-1214): "GONN", int32 version 1,
 * int32 tensor count, then per tensor int32 name length, name, int32 rank,
 * int32 shape[rank], int32 length, float32 data (little endian).  Tensors
 * are each layer's NamedParams (or its flat Params) named
 * layer_<i>_<ExtractLayerConfig type>_<name> (net.go:1425-1505). */
int gn_model_save_binary_weights(gn_model *m, const char *path);
/* Reads a SaveBinaryWeights file into this model's parameters and
 * BatchNorm2D running statistics; every tensor's name and length must match.
 * (The reference writes the format but has no reader.) */
int gn_model_load_binary_weights(gn_model *m, const char *path);
/* Network.SaveGGUF / SaveGGUFExt (net.go:1217-1392, gguf.go): GGUF v3 with
 * F32 tensors (f16 = 0) or F16 (f16 = 1, Float32ToFloat16's truncation). */
int gn_model_save_gguf(gn_model *m, const char *path, int32_t f16);
/* The whole training state for resume: parameters, Adam moments and
 * timestep, BatchNorm2D running statistics, MoE noise stream states.  No
 * counterpart in the reference, whose gob Save (net.go:863-1006) keeps no
 * Adam moments. */
int gn_model_save_state(gn_model *m, const char *path);
int gn_model_load_state(gn_model *m, const char *path);
/* Network.Save (net.go:863-871, Encode :1008-1075): "GONN", int32 1, then a
 * gob stream of int32(layers), the loss name, "Adam", one LayerConfig per
 * layer (ExtractLayerConfig, net.go:1393-1505), the flat parameters and
 * Adam's GobState (opt.go:262-322: its moments only when the network has at
 * most 1000 parameters, opt.go:129-153).  Byte for byte what a Go process
 * writes when Save is its first use of gob (gob numbers types per process). */
int gn_model_save_gob(gn_model *m, const char *path);
/* net.Load (net.go:875-1005): the reference's checks (magic, version, at
 * most 1000 layers, at most 256M parameters, the parameter count), then its
 * layers rebuilt with their saved parameters, value activations, the saved
 * loss and a fresh Adam(0.001) (the reference never restores the saved
 * optimizer state).  in_len is the input length per sample, needed when the
 * first layer is not Dense or Dropout (0 = from the file).  loss_kind
 * receives GN_LOSS_*.  Layer types, losses and optimizers this library does
 * not build are GN_ERR_UNSUPPORTED, as is a saved parameter count that
 * differs from the layer its config describes. */
int gn_model_load_gob(gn_ctx *ctx, const char *path, int32_t in_len, int32_t max_batch, int32_t workers,
                      gn_model **out, int32_t *loss_kind);

/* ---- per-layer operators on device pointers -----------------------------
 * Batched stand-ins for the per-sample Layer.Forward / Backward calls and the
 * Metal entry points listed next to each. */

/* matMulFusedPersistent + bias_activation (metal_ops.m:1235-1249, 171-195) /
 * Dense.ForwardWithArena (layer.go:346-456): out[b,o] = act(b[o] + x[b,:].W[o,:]).
 * Softmax/LogSoftmax pointers apply the row activation. */
int gn_dense_forward(gn_ctx *ctx, const float *x, const float *W, const float *bias, float *out,
                     int32_t B, int32_t in, int32_t out_n, int32_t act, int32_t act_is_ptr);
/* Dense.Backward (layer.go:488-667) for a batch: dz from gout and the saved
 * output, gradW = scale*dz^T x, gradB = scale*colsum(dz) (overwrite), and
 * gin = dz W when gin != NULL. */
int gn_dense_backward(gn_ctx *ctx, const float *x, const float *W, const float *out,
                      const float *gout, float *gradW, float *gradB, float *gin, float *dz_scratch,
                      int32_t B, int32_t in, int32_t out_n, int32_t act, int32_t act_is_ptr,
                      float scale);
/* No counterpart in the reference: gn_dense_backward for callers that cannot
 * allocate device memory (code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc).  Same arguments without the dz workspace;
 * dz and the partial sums live in a static 32 MiB device array of the
 * library (one per GPU, held until the process ends), so B x out_n may not
 * exceed 4,194,304 floats (GN_ERR_INVALID otherwise).  The call allocates
 * nothing.  Calls that overlap on one GPU share that array and race: the
 * caller serialises them. */
int gn_dense_backward_noalloc(gn_ctx *ctx, const float *x, const float *W, const float *out,
                              const float *gout, float *gradW, float *gradB, float *gin, int32_t B,
                              int32_t in, int32_t out_n, int32_t act, int32_t act_is_ptr, float scale);

/* Common to the operators below: B samples, each in the layer's flat
 * per-sample layout (its InSize / OutSize), row-major; parameter gradients
 * are written, not accumulated, and multiplied by `scale` (1/B gives the
 * batch average of Network.TrainBatch); an input gradient is written when its
 * pointer is not NULL.  Calls queue work on the context's stream. */

/* Conv2D.ForwardWithArena (conv2d.go:716-960, Metal conv path metal.go:6-50):
 * out = act(conv(x, W) + b) per sample, NCHW, params = [W (outC x inC x k x k)
 * | b (outC)] as Conv2D.Params().  act: scalar GN_ACT_* (Softmax not allowed). */
int gn_conv2d_forward(gn_ctx *ctx, const float *x, const float *params, float *out, int32_t B,
                      int32_t inC, int32_t H, int32_t W, int32_t outC, int32_t k, int32_t stride,
                      int32_t pad, int32_t act);
/* Conv2D.Backward (conv2d.go:997-1236) over the batch: dz = gout * act'(out),
 * grads = [dW | db] = scale * batch sums, gin = col2im(W^T dz). */
int gn_conv2d_backward(gn_ctx *ctx, const float *x, const float *params, const float *out,
                       const float *gout, float *grads, float *gin, int32_t B, int32_t inC,
                       int32_t H, int32_t W, int32_t outC, int32_t k, int32_t stride, int32_t pad,
                       int32_t act, float scale);
/* MaxPool2D.ForwardWithArena (maxpool2d.go:106-226; MaxPool2DPersistent
 * metal.go:343): first strict maximum of each window, padding never wins;
 * argmax = the winner's flat index inside its sample (int32, one per output). */
int gn_maxpool2d_forward(gn_ctx *ctx, const float *x, float *out, int32_t *argmax, int32_t B,
                         int32_t C, int32_t H, int32_t W, int32_t k, int32_t stride, int32_t pad);
/* MaxPool2D.Backward (maxpool2d.go:357-411): gin[i] = sum of gout over the
 * outputs whose argmax is i (every gin element is written). */
int gn_maxpool2d_backward(gn_ctx *ctx, const float *gout, const int32_t *argmax, float *gin,
                          int32_t B, int32_t C, int32_t H, int32_t W, int32_t k, int32_t stride,
                          int32_t pad);
/* Dropout.ForwardWithArena (dropout.go:85-155): in training mode mask (n
 * floats) receives the first n draws of RNG(42) against p (Reset reseeds the
 * stream before every sample, dropout.go:399-401, so every sample shares it)
 * and out = x * mask / (1 - p); in inference mode out = x. */
int gn_dropout_forward(gn_ctx *ctx, const float *x, float *out, float *mask, int32_t B, int32_t n,
                       float p, int32_t training);
/* Dropout.Backward (dropout.go:241-293): gin = gout * mask / (1 - p) in
 * training mode, gout otherwise. */
int gn_dropout_backward(gn_ctx *ctx, const float *gout, const float *mask, float *gin, int32_t B,
                        int32_t n, float p, int32_t training);
/* Output layer and loss: zo (B x C pre-activations) receives act(zo) (Softmax
 * / LogSoftmax rows when act_is_ptr, layer.go:183-205), loss_rows the
 * per-sample loss (MSE / CrossEntropy Forward, loss.go:53-70, 120-145) and dz
 * the gradient at the pre-activations (loss BackwardInPlace loss.go:91-112,
 * 165-185, then Dense's activation backward layer.go:488-567, Softmax
 * Jacobian included). */
int gn_softmax_ce_backward(gn_ctx *ctx, float *zo, const float *y, float *dz, float *loss_rows,
                           int32_t B, int32_t C, int32_t act, int32_t act_is_ptr, int32_t loss_kind);
/* LayerNorm.ForwardWithArena (layernorm.go:193-306) over `rows` rows of N:
 * y = gamma (x - mean) / std + beta, std = sqrt(var + eps) (eps 0 selects
 * 1e-5); stats = (mean, std) per row, kept for the backward. */
int gn_layernorm_forward(gn_ctx *ctx, const float *x, const float *gamma, const float *beta,
                         float *y, float *stats, int32_t rows, int32_t N, float eps);
/* LayerNorm.Backward (layernorm.go:334-441): dx by the reference's formula
 * (its last term divides by N std^2), dgamma = scale * sum g * xhat, dbeta =
 * scale * sum g; work = rows x N floats of scratch (used where N > 2048). */
int gn_layernorm_backward(gn_ctx *ctx, const float *g, const float *x, const float *gamma,
                          const float *stats, float *dx, float *dgamma, float *dbeta, float *work,
                          int32_t rows, int32_t N, float scale);
/* MultiHeadAttention (transformer.go:277-776): x is B x T x D, params = [wQ |
 * wK | wV | wOut], each a Linear Dense (W D x D, b D).  work carries the
 * forward's saved state to the backward: gn_mha_workspace floats, the same
 * buffer and x for both calls.  Any T and head size: up to T = 128 and
 * 32-wide heads with a pair's rows in LDS, heads of up to 128 in kernels that
 * stage the other side's rows, wider heads through batched GEMMs over the
 * materialised B x heads x T x T scores (included in the workspace); B x heads
 * must not exceed 65535. */
int gn_mha_workspace(int32_t B, int32_t T, int32_t D, int32_t heads, int32_t use_rope,
                     int64_t *floats);
/* MultiHeadAttention.ForwardWithArena (transformer.go:405-529): Q, K, V per
 * token, RoPE on Q and K when use_rope (applyRoPE transformer.go:212-236),
 * softmax(Q K^T / sqrt(hd)) V per head (causal mask -1e9), out = wOut(O). */
int gn_mha_forward(gn_ctx *ctx, const float *x, const float *params, float *out, float *work,
                   int32_t B, int32_t T, int32_t D, int32_t heads, int32_t causal, int32_t use_rope);
/* MultiHeadAttention.Backward (transformer.go:557-690): each projection's
 * weight gradient uses its last token's input (the per-token Dense layers
 * keep only the last Forward's input) and its bias gradient sums every
 * token; conjugate rotation before wQ / wK; gin = sum of the three
 * projections' input gradients. */
int gn_mha_backward(gn_ctx *ctx, const float *x, const float *params, const float *gout,
                    float *grads, float *gin, float *work, int32_t B, int32_t T, int32_t D,
                    int32_t heads, int32_t causal, int32_t use_rope, float scale);
/* SequenceUnroller(LSTM) with return_sequences false (unroller.go:57-213,
 * lstm.go:144-753): x is B x T x I, params = [Wx (4H x I) | Wh (4H x H) | b
 * (4H)], gates i, f, g, o; out = h_{T-1} (B x H); hidden <= 1024.  work:
 * gn_lstm_workspace floats (the same B, T, I, H, workers for both calls). */
int gn_lstm_workspace(int32_t B, int32_t T, int32_t I, int32_t H, int32_t workers,
                      int64_t *floats);
/* LSTM.ForwardWithArena per step (lstm.go:276-442): only the input gate adds Wx x +
 * Wh h to its bias (lstmComputeInputGates, lstm.go:1065-1101). */
int gn_lstm_seq_forward(gn_ctx *ctx, const float *x, const float *params, float *out, float *work,
                        int32_t B, int32_t T, int32_t I, int32_t H, int32_t return_sequences);
/* SequenceUnroller.Backward + LSTM.Backward per step (unroller.go:133-213,
 * lstm.go:476-699, clipGradients 725-753): carried dh (dh_{t-1} = dh_t + Wh^T dG), dWx from the last
 * step's input, each worker chain's cumulative gradient clipped to norm 1
 * after every step (`workers` chains of ceil(B / workers) samples, as
 * trainBatchParallel's chunks), gin_t = Wx^T dG_t (unclipped).  return_sequences
 * (NewSequenceUnroller's flag, unroller.go:21-43): out / gout hold every step's
 * h (B x T x H) instead of the last (B x H). */
int gn_lstm_seq_backward(gn_ctx *ctx, const float *x, const float *params, const float *gout,
                         float *grads, float *gin, float *work, int32_t B, int32_t T, int32_t I,
                         int32_t H, int32_t workers, float scale, int32_t return_sequences);
/* Embedding.ForwardWithArena (embedding.go:79-141): x = B x T ids as floats,
 * out = rows of E (V x D), ids = the int32 indices for the backward; bad
 * (optional, B ints) = 1 for a sample with an id outside [0, V), which the
 * reference's Forward rejects (its output rows read row 0 here). */
int gn_embedding_forward(gn_ctx *ctx, const float *x, const float *E, float *out, int32_t *ids,
                         int32_t *bad, int32_t B, int32_t T, int32_t V, int32_t D);
/* Embedding.Backward (embedding.go:147-183) over a batch: Backward zeroes the
 * table's gradient before adding a sample's rows, so gradE = scale * the rows
 * of the last sample of each worker chunk (`workers` chunks of ceil(B /
 * workers); with bad, the last sample the reference's loop still reaches).
 * Contributing rows (chunks x T) above 2048 take a list in the context's
 * scratch (2 ints per row; GN_ERR_UNSUPPORTED beyond 8M rows). */
int gn_embedding_backward(gn_ctx *ctx, const float *gout, const int32_t *ids, const int32_t *bad,
                          float *gradE, int32_t B, int32_t T, int32_t V, int32_t D, int32_t workers,
                          float scale);

/* AvgPool2D.ForwardWithArena / Backward (avgpool2d.go:137-474): B samples of
 * C x H x W, k x k windows, stride, zero padding not counted in the mean. */
int gn_avgpool2d_forward(gn_ctx *ctx, const float *x, float *out, int32_t B, int32_t C, int32_t H,
                         int32_t W, int32_t k, int32_t stride, int32_t pad);
int gn_avgpool2d_backward(gn_ctx *ctx, const float *gout, float *gin, int32_t B, int32_t C, int32_t H,
                          int32_t W, int32_t k, int32_t stride, int32_t pad);
/* RMSNorm.ForwardWithArena / Backward (rmsnorm.go:222-329) over `rows` rows of
 * N: y = gamma x / rms, rms per row for the backward (eps 0 selects 1e-5);
 * dx (may be NULL) follows the reference's formula; dgamma = scale * sums;
 * work: rows x N floats of scratch (used where N > 2048). */
int gn_rmsnorm_forward(gn_ctx *ctx, const float *x, const float *gamma, float *y, float *rms,
                       int32_t rows, int32_t N, float eps);
int gn_rmsnorm_backward(gn_ctx *ctx, const float *g, const float *x, const float *gamma, const float *rms,
                        float *dx, float *dgamma, float *work, int32_t rows, int32_t N, float scale);
/* SwiGLU.ForwardWithArena / Backward (swiglu.go:103-232): params = [W | V]
 * (out x in each, no biases), y = swish(W x) * (V x); grads = [dW | dV]
 * written (scale * sums); gin may be NULL; work: gn_swiglu_workspace floats
 * shared by the forward and backward of one batch. */
int gn_swiglu_workspace(int32_t B, int32_t out, int64_t *floats);
int gn_swiglu_forward(gn_ctx *ctx, const float *x, const float *params, float *out, float *work, int32_t B,
                      int32_t in, int32_t out_size);
int gn_swiglu_backward(gn_ctx *ctx, const float *x, const float *params, const float *gout, float *grads,
                       float *gin, float *work, int32_t B, int32_t in, int32_t out_size, float scale);
/* BatchNorm2D.ForwardWithArena / Backward (batchnorm2d.go:255-666): B samples
 * of C x HW; params = [gamma | beta] or NULL (affine = false).  training:
 * each sample normalised by its own channel statistics (the reference runs one
 * sample per Forward), running mean / var advanced once per sample in sample
 * order; stats = 3 B C floats (mean, var, std) for the backward.  Inference
 * uses the running statistics; its backward gives dx only and zero parameter
 * gradients (batchnorm2d.go:525-551).  work: 2 B C floats. */
int gn_batchnorm2d_forward(gn_ctx *ctx, const float *x, const float *params, float *out, float *stats,
                           float *running_mean, float *running_var, int32_t B, int32_t C, int32_t HW,
                           float eps, float momentum, int32_t training);
int gn_batchnorm2d_backward(gn_ctx *ctx, const float *gout, const float *x, const float *params,
                            const float *stats, const float *running_var, float *grads, float *gin,
                            float *work, int32_t B, int32_t C, int32_t HW, float eps, int32_t training,
                            float scale);
/* SequenceUnroller(GRU) forward / backward (unroller.go:57-213,
 * gru.go:192-703): x = B x T x I, params = [Wx (3H x I) | Wh (2H x H) | b
 * (3H)], the reference's quirks kept (candidate weighted by 1 - u in the
 * backward, no reset-gate delta, dWx from the last step's input, carried dh);
 * return_sequences: out / gout hold every step's h.  work: gn_gru_workspace
 * floats, shared by the forward and backward of one batch. */
int gn_gru_workspace(int32_t B, int32_t T, int32_t I, int32_t H, int64_t *floats);
int gn_gru_seq_forward(gn_ctx *ctx, const float *x, const float *params, float *out, float *work, int32_t B,
                       int32_t T, int32_t I, int32_t H, int32_t return_sequences);
int gn_gru_seq_backward(gn_ctx *ctx, const float *x, const float *params, const float *gout, float *grads,
                        float *gin, float *work, int32_t B, int32_t T, int32_t I, int32_t H, float scale,
                        int32_t return_sequences);
/* MoE.ForwardWithArena / Backward (moe.go:140-313): params = [gating W (E x
 * I), b | per expert W (O x I), b]; the top K experts by gate softmax
 * (stable in index order for ties), LeakyReLU(0.1) experts.  training adds
 * the layer's RNG gate noise: *noise is the stream's state (42 at
 * construction), advanced by E draws per sample; and the load-balancing
 * gradient.  work: gn_moe_workspace floats, shared by the forward and
 * backward of one batch. */
int gn_moe_workspace(int32_t B, int32_t I, int32_t O, int32_t E, int32_t K, int64_t *floats);
int gn_moe_forward(gn_ctx *ctx, const float *x, const float *params, float *out, float *work, int32_t B,
                   int32_t I, int32_t O, int32_t E, int32_t K, int32_t training, uint64_t *noise);
int gn_moe_backward(gn_ctx *ctx, const float *x, const float *params, const float *gout, float *grads,
                    float *gin, float *work, int32_t B, int32_t I, int32_t O, int32_t E, int32_t K,
                    int32_t training, float scale);

/* ---- answering token by token ---------------------------------------------
 * No counterpart in the reference, whose Predict runs the whole window for
 * every token.  A paged cache of rotated keys and values in 8 bits, the
 * attention that reads it, and the draw of the next token.  Device pointers;
 * calls queue work on the context's stream, allocate nothing and do not
 * synchronise (but gn_rope_tables); what lies in device memory (starts, lens,
 * the page table, settings) is read when the work runs.  Calls that may run at
 * the same time (two contexts) need a `work` each.  Like the other operators
 * they may use the context's scratch.
 *
 * Tokens are packed: sequence b's new tokens are the rows starts[b] ..
 * starts[b + 1] - 1 (starts: B + 1 int32) of the inputs and outputs, at the
 * positions lens[b], lens[b] + 1, ... (lens: B int32, the tokens cached before
 * the call; the caller advances it after the step).  A sequence may have no
 * new token; rows outside every sequence are neither read nor written.  B and
 * heads are 65535 at most, N and B * max_new 2^26, a sequence's tokens and B *
 * max_new * heads 2^31 - 4097. */
#define GN_DTYPE_F32 0
#define GN_DTYPE_BF16 1

/* The cache's memory, all of it the caller's.  Pages of page_size tokens (16,
 * 32, 64 or 128), head_dim 1 to 256.  Bytes are E4M3 (sign, 4 exponent, 3
 * mantissa bits; 0x7f NaN); a byte stands for its value times the power of two
 * in the scale of its page and head.  Position p of sequence b is token p %
 * page_size of page table[b * max_pages + p / page_size].  Zero a new cache's
 * k and v once (gn_memset_zero); scales need no start.  While a call
 * appends to a page, that page belongs to one sequence; full pages may stand
 * in several sequences' tables. */
typedef struct gn_kv_cache {
  void *k;              /* pages x kv_heads x page_size x row */
  void *v;              /* pages x kv_heads x row x page_size (transposed) */
  float *k_scale;       /* pages x kv_heads */
  float *v_scale;       /* pages x kv_heads */
  const int32_t *table; /* B x max_pages */
  int32_t pages, page_size, kv_heads, head_dim, max_pages;
} gn_kv_cache;
/* bytes of k (and of v) and the padded row: head_dim rounded up to 32, 64, 96,
 * 128, 192 or 256. */
int gn_kv_cache_bytes(int32_t pages, int32_t page_size, int32_t kv_heads, int32_t head_dim, int64_t *bytes,
                      int32_t *row);
/* applyRoPE's angles (transformer.go:212-236) of positions 0 .. positions - 1
 * for heads of head_dim, the same numbers as gn_mha_forward uses: cos and sin
 * are positions x (head_dim / 2) floats.  Synchronises. */
int gn_rope_tables(gn_ctx *ctx, float *cos, float *sin, int32_t positions, int32_t head_dim);
/* Rotates new queries and keys by their positions and appends keys and values
 * to the cache, one launch.  q: rows of heads x head_dim, k and v: rows of
 * kv_heads x head_dim, in dtype; strides in elements from one token's row to
 * the next (queries, keys and values may lie side by side in one matrix).  The
 * pair (x_i, x_{i + head_dim/2}) turns by (cos, sin)[position][i]; cos and sin
 * null: nothing turns.  q_out (may be q itself, with its stride) receives the
 * queries in dtype; q and q_out null: keys and values only.  N: rows of the
 * inputs; max_new: the largest number of new tokens of a sequence; rope_len:
 * positions in cos and sin.
 * The scale of a block (one page, one head, K or V apart) is the smallest power
 * of two, 2^-100 at least, that brings its finite values within 448, or the
 * block's scale so far if that is larger and the block holds tokens already;
 * where it grows, the tokens already there are scaled to it (exact but for what
 * falls below the smallest E4M3 step).  A rotated value is rounded to float32
 * and then to the nearest E4M3 value, ties to even; a value that is not finite
 * is kept as NaN.
 * bad (may be null; B int32, cleared by the caller): set to 1 for a sequence
 * that is skipped whole because its starts or lens lie outside [0, N] or the
 * table, it has more than max_new tokens or positions beyond rope_len, and for
 * one with a page outside [0, pages), whose tokens are not stored. */
int gn_kv_append(gn_ctx *ctx, const gn_kv_cache *kv, const void *q, const void *k, const void *v, void *q_out,
                 int64_t q_stride, int64_t k_stride, int64_t v_stride, int64_t q_out_stride, const float *cos,
                 const float *sin, int32_t rope_len, const int32_t *starts, const int32_t *lens, int32_t B, int32_t N,
                 int32_t max_new, int32_t heads, int32_t dtype, int32_t *bad);
/* out = softmax(scale q K^T) V over each sequence's cache, after its new
 * tokens were appended: a query at position p sees positions 0 .. p (causal) or
 * all of lens[b] + new tokens.  heads must be a multiple of kv_heads (query head
 * h reads key head h / (heads / kv_heads)).  q, out: N rows of heads x head_dim
 * in dtype.  max_len: an upper bound of lens[b] + new tokens, from which (with
 * max_new) the work is split; a sequence beyond it is skipped.  Sums and
 * maxima are float32; the products of float32 queries have float32's precision,
 * the weights of bfloat16 ones keep 16 bits.  Tokens in pages
 * outside [0, pages) are left out; a query that sees none gives 0.  A NaN that a
 * query sees, in its keys or values, makes its output NaN; one that it does not see
 * is nothing to it.  bad as above.  work: gn_kv_attention_workspace floats, 16-byte
 * aligned (may be 0: then work may be null).  What it asks for serves every call with the
 * same heads whose B, max_new and max_len are no larger, so that a program asks once for
 * its largest sizes, and gn_kv_attention_window's and gn_kv_attention_tree's as well. */
int gn_kv_attention_workspace(int32_t B, int32_t max_new, int32_t max_len, int32_t heads, int32_t kv_heads,
                              int32_t head_dim, int64_t *floats);
int gn_kv_attention(gn_ctx *ctx, const gn_kv_cache *kv, const void *q, void *out, int64_t q_stride,
                    int64_t out_stride, const int32_t *starts, const int32_t *lens, int32_t B, int32_t N,
                    int32_t max_new, int32_t max_len, int32_t heads, float scale, int32_t causal, int32_t dtype,
                    float *work, int32_t *bad);
/* gn_kv_attention for long streams: a query at position p sees the first `sinks` tokens
 * and the last `window` up to its own, p - window + 1 .. p.  Of both 0 a query sees
 * nothing and gives 0.  Pages that no query of the call sees may be gone: their entries
 * in the table may hold anything.  work: gn_kv_attention_workspace floats, as
 * gn_kv_attention's. */
int gn_kv_attention_window(gn_ctx *ctx, const gn_kv_cache *kv, const void *q, void *out, int64_t q_stride,
                           int64_t out_stride, const int32_t *starts, const int32_t *lens, int32_t B, int32_t N,
                           int32_t max_new, int32_t max_len, int32_t heads, float scale, int32_t sinks, int32_t window,
                           int32_t dtype, float *work, int32_t *bad);

/* Drafted tokens: a tree of guesses is appended, attended to and drawn for in one
 * step, and the path that turns out right is kept.
 * gn_kv_append for rows whose positions are not those of their places: the token of row r
 * is stored as its sequence's next one as gn_kv_append stores it, and it and its query turn
 * by (cos, sin)[positions[r]] (positions: N int32 on the device; two guesses for one place
 * have one position).  A position outside [0, rope_len) makes the row's query and key NaN
 * and flags its sequence.  Without cos and sin positions may be null. */
int gn_kv_append_at(gn_ctx *ctx, const gn_kv_cache *kv, const void *q, const void *k, const void *v, void *q_out,
                    int64_t q_stride, int64_t k_stride, int64_t v_stride, int64_t q_out_stride, const float *cos,
                    const float *sin, int32_t rope_len, const int32_t *positions, const int32_t *starts,
                    const int32_t *lens, int32_t B, int32_t N, int32_t max_new, int32_t heads, int32_t dtype,
                    int32_t *bad);
/* gn_kv_attention of new tokens that see all lens[b] cached ones and, of their sequence's
 * new ones, those that a mask names: bit j % 32 of word j / 32 of row r (mask: N rows,
 * mask_stride words apart, of a bit for each of up to max_new tokens) says that the token
 * of row r sees its sequence's j-th new token.  Its own bit is like any other; bits behind
 * the sequence's new tokens are not looked at.  work: gn_kv_attention_workspace floats. */
int gn_kv_attention_tree(gn_ctx *ctx, const gn_kv_cache *kv, const void *q, void *out, int64_t q_stride,
                         int64_t out_stride, const uint32_t *mask, int64_t mask_stride, const int32_t *starts,
                         const int32_t *lens, int32_t B, int32_t N, int32_t max_new, int32_t max_len, int32_t heads,
                         float scale, int32_t dtype, float *work, int32_t *bad);
/* Keeps counts[b] (B int32) of a sequence's new tokens: the keep[starts[b] + i]-th
 * becomes the i-th, i < counts[b]; their numbers rise (keep: N int32, those behind the
 * counts are not looked at).  The caller advances lens[b] by counts[b].  Where tokens
 * move into a block (one page, one head, K or V apart), its scale becomes the largest of its
 * own and those of the blocks they come from, and all bytes of the block are scaled to it
 * (exact but for what falls below the smallest E4M3 step).  The pages of the new tokens
 * belong to one sequence.  bad as above: set for a sequence that is skipped whole because
 * its bounds, counts or numbers are wrong or a page is outside [0, pages). */
int gn_kv_keep(gn_ctx *ctx, const gn_kv_cache *kv, const int32_t *keep, const int32_t *counts, const int32_t *starts,
               const int32_t *lens, int32_t B, int32_t N, int32_t max_new, int32_t *bad);
/* MultiHeadAttention (transformer.go:405-529) for new tokens of B sequences
 * over such a cache: x and out are N rows of D floats, params as
 * gn_mha_forward's; Q, K, V of the new tokens, rotated where cos and sin are
 * given (gn_rope_tables), K and V appended, causal attention over the cache, wOut.
 * kv->kv_heads x kv->head_dim must be D.  With all tokens at once and empty sequences it
 * computes gn_mha_forward's causal layer, keys and values rounded to 8 bits.  A sequence
 * beyond max_len, the table or rope_len is neither appended nor attended to.  Rows
 * outside every sequence, and of a sequence that is skipped, get wOut's bias.  work:
 * gn_mha_cached_workspace floats for B, N, max_new and max_len as large or larger. */
int gn_mha_cached_workspace(int32_t B, int32_t N, int32_t max_new, int32_t max_len, int32_t D, int32_t heads,
                            int64_t *floats);
int gn_mha_cached_forward(gn_ctx *ctx, const gn_kv_cache *kv, const float *x, const float *params, float *out,
                          const float *cos, const float *sin, int32_t rope_len, const int32_t *starts,
                          const int32_t *lens, int32_t B, int32_t N, int32_t max_new, int32_t max_len, int32_t D,
                          float *work, int32_t *bad);
/* Rules for B rows of V logits, all arrays on the device; a null pointer leaves its rule
 * out.  Row b's text is the first token_lens[b] of tokens[b * tokens_stride ..] (null: all
 * tokens_stride), the first prompt_lens[b] of them (null: none) the prompt; its biases the
 * first bias_lens[b] (null: all) of bias_ids and bias [b * bias_stride ..].  Lengths below 0
 * count as 0, above the stride as the stride, ids outside [0, V) as none.  Row
 * allowed_row[b] (null: b) of `allowed`, allowed_stride words of 32 tokens, lowest bit
 * first, names the tokens that may follow; a number outside [0, allowed_rows): all may. */
typedef struct gn_logit_rules {
  const float *repetition, *frequency, *presence; /* B each */
  const int32_t *tokens, *token_lens, *prompt_lens;
  int64_t tokens_stride;
  const int32_t *bias_ids;
  const float *bias;
  const int32_t *bias_lens;
  int64_t bias_stride;
  const uint32_t *allowed;
  const int32_t *allowed_row;
  int64_t allowed_stride;
  int32_t allowed_rows;
} gn_logit_rules;
/* out (may be logits itself, with their stride) = the logits under the rules, for
 * gn_sample.  In this order, in float32: a token of the text has a logit above 0 divided by
 * repetition[b], any other multiplied by it (a repetition that is not above 0 counts as 1);
 * one that stands n > 0 times behind the prompt loses frequency[b] n and then presence[b];
 * one with a bias gains it (of several the last entry's); one that may not follow becomes
 * -inf, whatever it was.  Rows may be anything that gn_sample takes.  V <= 2^20, lists of a
 * row <= 2^30. */
int gn_logits_adjust(gn_ctx *ctx, const void *logits, int64_t stride, void *out, int64_t out_stride, int32_t dtype,
                     const gn_logit_rules *rules, int32_t B, int32_t V);
/* Draws one index of each of B rows of V logits (row stride in elements, dtype)
 * with the given random number u[b] in [0, 1).  With m the row's largest logit,
 * w_i = exp((z_i - m) / temperature[b]); NaN and -inf logits are left out.  Kept
 * are the top_k[b] largest logits (<= 0: all), of those the shortest run in
 * falling order whose weights reach top_p[b] of their sum (>= 1: all, <= 0: the
 * first), of those the ones with w_i >= min_p[b]; the largest always stays, and
 * equal logits go by the lowest index.  ids[b] is the first index, in rising
 * order, at which the kept weights' running sum exceeds u[b] times their sum; -1
 * for a row without a logit to choose.  A temperature that is not above 0 takes
 * the largest logit; beside an infinite logit finite ones weigh nothing.  A top_p
 * that is NaN keeps all, a min_p that is NaN the largest.  All settings are device
 * arrays of B; temperature (1), top_k, top_p and min_p may be null.  Weights are
 * float64 exponentials rounded to whole multiples of 2^-43 and summed as integers,
 * so a result does not depend on any order of sums.  V <= 2^20.  work: gn_sample_workspace floats
 * for V and as many rows or more, 8-byte aligned. */
int gn_sample_workspace(int32_t B, int32_t V, int64_t *floats);
int gn_sample(gn_ctx *ctx, const void *logits, int64_t stride, int32_t dtype, const float *temperature,
              const int32_t *top_k, const float *top_p, const float *min_p, const float *u, int32_t *ids, int32_t B,
              int32_t V, float *work);

/* Generic fp32 GEMM: C[M,N] = alpha * op(A) op(B); trans flags as BLAS
 * (A is M x K row-major when transA == 0, K x M when 1; B is K x N when
 * transB == 0, N x K when 1).  On fp32 MFMA; large ones with K a multiple of
 * 64 from 320 on as six bf16 MFMA products of the operands' exact three-way
 * split, with a smaller error over all of float32's range.  Stands in for
 * matMulMPSPersistent (metal_ops.m:1220-1233). */
int gn_gemm(gn_ctx *ctx, int32_t transA, int32_t transB, int32_t M, int32_t N, int32_t K,
            float alpha, const float *A, int32_t lda, const float *B, int32_t ldb, float *C,
            int32_t ldc);
/* Adam.StepInPlace (opt.go:207-252) over n elements of the flat arena, with
 * the optimizer timestep already advanced (first Network.Step => 1). */
int gn_adam_step(gn_ctx *ctx, float *params, const float *grads, float *m, float *v, int64_t n,
                 float lr, float beta1, float beta2, float eps, int32_t timestep);

/* ---- kernel timing (measurement hook; no reference counterpart) ---------
 * While enabled, every kernel launch of the library is bracketed by HIP events
 * on the context stream and attributed to a class.  gn_timing_report
 * synchronises the stream and returns the launch count and summed kernel time
 * of a class since the last enable. */
#define GN_KCLASS_GEMM 0   /* gemm_f32_mfma (Dense fwd / dX / dW) */
#define GN_KCLASS_ADAM 1   /* adam_kernel */
#define GN_KCLASS_OTHER 2  /* row kernels, column sums, dropout, ... */
int gn_timing_enable(gn_ctx *ctx, int enable);
int gn_timing_report(gn_ctx *ctx, int kclass, int64_t *launches, double *total_ms);
/* Per kernel (or fused launch group) since the last enable: name, class,
 * launch count, summed time and summed algorithmic work -- bytes moved for a
 * memory-bound kernel (compulsory fp32 reads and writes), FLOPs for a GEMM /
 * matrix-core kernel -- so units / time is its achieved GB/s or FLOP/s.
 * Writes at most cap entries and the number of distinct names to *n. */
typedef struct gn_kernel_stat {
  char name[48];
  int32_t cls;      /* GN_KCLASS_* */
  int64_t launches;
  double ms;
  double units;
} gn_kernel_stat;
int gn_timing_kernels(gn_ctx *ctx, gn_kernel_stat *out, int32_t cap, int32_t *n);
/* The launch floor the per-kernel times are read against: reps launches of an
 * empty kernel of `blocks` 256-thread workgroups on the context stream, timed
 * like every library launch (recorded as "floor" while timing is enabled). */
int gn_timing_floor(gn_ctx *ctx, int32_t blocks, int32_t reps);

/* ---- synthetic inputs (host side; harness utility) ----------------------
 * The reference's LCG (layer.go:61-81): U[0,1) stream, N(0,1) by one
 * Box-Muller cosine per two draws (u1 clamped to 1e-7, f64 math), class ids
 * floor(U*nclass) clamped to nclass-1. */
int gn_fill_uniform(float *dst, int64_t n, uint64_t seed);
int gn_fill_normal(float *dst, int64_t n, uint64_t seed);
int gn_fill_class_ids(int32_t *dst, int64_t n, int32_t nclass, uint64_t seed);

#ifdef __cplusplus
}
#endif
#endif /* GONEURON_HIP_H */
