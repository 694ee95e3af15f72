/*
 * mmfe — MI355X (gfx950) signal front-end, C ABI.
 *
 * The reference (lixinghe1999/multi_modal) is pure Python and has no FFI of its own: the
 * boundary it offers for this path is a set of Python call sites that hand a waveform to a
 * third-party CPU routine.  Each entry point below names the call site(s) it stands behind;
 * the Python wrappers in multi_modal_amd/ keep those call signatures and bind this library
 * with ctypes.
 *
 *   kind MMFE_KIND_FBANK     torchaudio.compliance.kaldi.fbank(...) called from
 *                            classification/vggsound/dataset/vggsound.py:45-47, with the
 *                            pad/cut to 384 frames and the affine normalisation of
 *                            vggsound.py:48-59 fused in (out_frames / pad_value / out_shift /
 *                            out_scale).
 *   kind MMFE_KIND_LOGSPEC   librosa.stft(...) + np.log(|X|^2 + eps) of
 *                            classification/recognition/dataset/epic_kitchen.py:114-126 and
 *                            classification/retrieval/dataset/epic_kitchen.py:141-153, with the
 *                            /255 of classification/recognition/dataset/transform.py:268-285
 *                            fused in (out_scale).  Also serves the long-utterance log-mel
 *                            configuration (centre reflect padding, mel, log10, per-clip clamp).
 *   kind MMFE_KIND_STFT_MAG  np.abs(scipy.signal.stft(x, fs, nperseg, noverlap)[-1]) of
 *                            classification/har/adbox.py:20.
 *   kind MMFE_KIND_FRAME     frame_signal(signal, frame_length, hop_length, window) of
 *                            classification/vggsound/utils/transforms.py:19-61 (identical copies
 *                            under recognition/ and retrieval/).
 *   kind MMFE_KIND_RESAMPLE  the sample-rate conversion in front of the path: librosa.load(file,
 *                            sr=16000, duration=10) of classification/vggsound/dataset/vggsound.py:114
 *                            and ffmpeg -ar 24000 of
 *                            classification/recognition/dataset/extract_audio.py:6-13 (filter design,
 *                            alignment and output length of scipy.signal.resample_poly).
 *
 * Conventions
 *   - Every function returns 0 on success and a negative MMFE_E* code on failure; the message is
 *     available from mmfe_last_error() (thread-local).  Nothing throws across the ABI, nothing
 *     calls exit().
 *   - All data pointers passed to mmfe_run* are DEVICE pointers owned by the caller (e.g.
 *     tensor.data_ptr()).  The library allocates only plan-lifetime constant tables.
 *   - Input samples are float32, or (spec.in_dtype = MMFE_IN_S16) the signed 16-bit PCM the reference's audio
 *     files hold, decoded in the kernel's loads; strides and offsets always count input elements.
 *   - mmfe_run* is asynchronous on the given HIP stream (NULL = the default stream); it never
 *     synchronises and never allocates.
 *   - Plans are immutable after creation and may be shared between threads and streams, with one
 *     exception: a plan with clamp_below_max > 0 owns a per-row scratch (row maxima and minima), so
 *     two mmfe_run* calls on such a plan must not overlap on the device (issue them on one stream, or
 *     create one plan per stream); a call handles at most 2^20 rows.
 *   - There is no CPU path: creating a plan without a usable gfx950 device fails.
 */
#ifndef MMFE_H
#define MMFE_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MMFE_ABI_VERSION 7

/* error codes */
#define MMFE_OK            0
#define MMFE_EINVAL       -1   /* bad argument / unsupported parameter combination */
#define MMFE_ENODEVICE    -2   /* no usable HIP device */
#define MMFE_EHIP         -3   /* a HIP runtime call failed */
#define MMFE_ENOMEM       -4

/* mmfe_spec.kind */
#define MMFE_KIND_FBANK     1
#define MMFE_KIND_LOGSPEC   2
#define MMFE_KIND_STFT_MAG  3
#define MMFE_KIND_FRAME     4
#define MMFE_KIND_RESAMPLE  5  /* rational-ratio polyphase FIR resampler: rows of n samples -> rows of ceil(n * up / down) samples.
                                  Stands where the reference resamples on the CPU before anything else happens:
                                  librosa.load(file, sr=16000, duration=10) (classification/vggsound/dataset/vggsound.py:114) and
                                  ffmpeg -ar 24000 (classification/recognition/dataset/extract_audio.py:6-13).
                                  Fields: n_fft = up, hop = down (coprime), win_len = number of FIR taps (odd), `window` = the taps
                                  (low-pass of cutoff 1/max(up, down), already multiplied by up), out_frames = 0 or the number of
                                  output samples rows are cut / zero-padded to (duration=...), in_dtype float32 or 16-bit PCM;
                                  every other field 0 / MMFE_*_NONE.  Alignment, output count and edge handling (zeros beyond the
                                  row) are those of scipy.signal.resample_poly(x, up, down).  Output: (n_rows, samples), float32 */

/* mmfe_spec.pad_mode: how samples outside [0, n) are read */
#define MMFE_PAD_NONE     0    /* never read outside (snip-edges framing) */
#define MMFE_PAD_ZERO     1
#define MMFE_PAD_REFLECT  2

/* mmfe_spec.frames_mode: number of frames for an n-sample row */
#define MMFE_FRAMES_SNIP    0  /* n < win_len ? 0 : 1 + (n - win_len) / hop          (kaldi snip_edges) */
#define MMFE_FRAMES_CENTER  1  /* 1 + n / hop, frame t centred on sample t*hop        (librosa center=True) */
#define MMFE_FRAMES_SCIPY   2  /* 1 + ceil(n / hop), zero-extended by win_len/2       (scipy boundary='zeros', padded) */
#define MMFE_FRAMES_CEIL    3  /* n <= win_len ? 1 : 1 + ceil((n - win_len) / hop), zero pad split floor/ceil (frame_signal) */

/* mmfe_spec.log_kind */
#define MMFE_LOG_NONE       0
#define MMFE_LOG_LN_MAX     1  /* ln(max(x, log_floor))      kaldi */
#define MMFE_LOG_LN_ADD     2  /* ln(x + log_floor)          EPIC  */
#define MMFE_LOG_LOG10_MAX  3  /* log10(max(x, log_floor))   long-utterance log-mel */

/* mmfe_spec.layout */
#define MMFE_LAYOUT_TIME_MAJOR  0  /* out[row][frame][feature] */
#define MMFE_LAYOUT_FEAT_MAJOR  1  /* out[row][feature][frame] */

/* mmfe_spec.out_dtype: element type of the output tensor */
#define MMFE_OUT_F32   0
#define MMFE_OUT_F16   1  /* IEEE half, round to nearest even: what the encoders' @autocast() casts the spectrogram to
                           (classification/vggsound/models/vit_model.py:388); FBANK and LOGSPEC kinds (the any-length DFT kernel not
                           together with clamp_below_max) */
#define MMFE_OUT_BF16  2  /* bfloat16, round to nearest even; same kinds */

/* mmfe_spec.in_dtype: element type of the input rows */
#define MMFE_IN_F32   0
#define MMFE_IN_S16   1  /* signed 16-bit PCM, sample value = s / 32768 (exact in float32): what torchaudio.load
                           (classification/vggsound/dataset/vggsound.py:66) and librosa.load
                           (classification/recognition/dataset/epic_kitchen.py:135) make of the 16-bit FLAC / pcm_s16le
                           WAV files the reference stores (vggsound.py:120, recognition/dataset/extract_audio.py:9);
                           FBANK, LOGSPEC and RESAMPLE kinds */
#define MMFE_IN_F64   2  /* FRAME kind only: frame_signal multiplies in the dtype of its operands
                           (classification/vggsound/utils/transforms.py:24-25, 58-59), so float64 rows take a float64 window
                           (spec.window_f64 = 1) and give float64 frames, one correctly rounded product each */
#define MMFE_IN_F16   3  /* FRAME kind only: IEEE half rows, float window holding half values, half frames (the exact product
                           rounded once to nearest even, as torch multiplies halves) */
#define MMFE_IN_BF16  4  /* FRAME kind only: bfloat16 rows, likewise */

typedef struct mmfe_spec {
    int32_t struct_size;   /* = sizeof(mmfe_spec) */
    int32_t kind;          /* MMFE_KIND_* */
    int32_t n_fft;         /* DFT length in [2, 4096]; 512, 400 and (STFT_MAG) 32 have radix kernels.  Other lengths run on the
                              any-length kernel, which needs 32*n_fft + 128*(win_len + 1) bytes of LDS (plus 64*(n_fft/2 + 2) when
                              n_fft > 510): plans beyond the CU's 160 KiB (win_len near n_fft above about 850) are refused at creation */
    int32_t win_len;       /* number of window taps (<= n_fft); FRAME: frame_length */
    int32_t win_off;       /* position of tap 0 inside the n_fft-long DFT input (zeros elsewhere) */
    int32_t hop;
    int32_t pad_mode;      /* MMFE_PAD_* */
    int32_t frames_mode;   /* MMFE_FRAMES_* */
    int32_t n_mel;         /* 0 = no mel projection, features are the n_fft/2+1 DFT bins */
    int32_t remove_dc;     /* subtract the per-frame mean before pre-emphasis (kaldi) */
    float   preemph;       /* 0 = off; y[j] = x[j] - preemph * x[max(j-1,0)] */
    int32_t power;         /* 1 = |X|, 2 = |X|^2 */
    float   spec_scale;    /* multiplies X before |.| (scipy 'spectrum' scaling = 1/sum(window)); 1 = off */
    int32_t log_kind;      /* MMFE_LOG_* */
    float   log_floor;
    float   out_shift;     /* result = (value + out_shift) * out_scale */
    float   out_scale;
    int32_t out_frames;    /* 0 = natural frame count; else rows are cut / padded to this many frames */
    float   pad_value;     /* value (before shift/scale) of padded frames */
    int32_t drop_last;     /* drop the last natural frame (long-utterance log-mel) */
    float   clamp_below_max; /* > 0: per-row clamp to (row max - clamp_below_max) before shift/scale */
    int32_t layout;        /* MMFE_LAYOUT_* */
    int32_t window_f64;    /* 1: the `window` argument of mmfe_plan_create points to doubles (librosa / scipy build
                              their windows in float64 and multiply in float64); 0: floats */
    int32_t out_dtype;     /* MMFE_OUT_*: the arithmetic stays float32, only the stored value is rounded */
    int32_t in_dtype;      /* MMFE_IN_*: 16-bit PCM results are bit-identical to running on the decoded float32 samples; the FRAME
                              kind stores frames of its rows' own type */
} mmfe_spec;

typedef struct mmfe_plan mmfe_plan;

/* Library / ABI version (MMFE_ABI_VERSION of the build). */
int mmfe_abi_version(void);

/* Last error message of the calling thread ("" if none). */
const char* mmfe_last_error(void);

/* Number of usable devices (0 when there is none; never fails). */
int mmfe_device_count(void);

/* Output shape for rows of n_samples samples: number of frames and features per frame.
 * Pure host arithmetic, no device needed.
 * Stands for the shape rules of kaldi snip-edges framing, librosa centred framing,
 * scipy.signal.stft and frame_signal (transforms.py:32-37). */
int mmfe_spec_out_shape(const mmfe_spec* spec, int64_t n_samples, int64_t* n_frames, int64_t* n_feat);

/* Build a plan: validates the spec, uploads the constant tables to `device`.
 *   window        host, win_len floats (doubles when spec->window_f64), the values exactly as the
 *                 reference library builds them
 *   band_start    host, n_mel ints: first DFT bin of each mel filter          (NULL when n_mel == 0)
 *   band_len      host, n_mel ints: number of consecutive bins of each filter (0 allowed)
 *   band_weights  host, sum(band_len) floats, filter after filter
 * Replaces the per-call table construction inside kaldi.fbank / librosa.stft / scipy.signal.stft. */
int mmfe_plan_create(const mmfe_spec* spec, const void* window,
                     const int32_t* band_start, const int32_t* band_len, const float* band_weights,
                     int device, mmfe_plan** out_plan);

int mmfe_plan_destroy(mmfe_plan* plan);

/* Run the transform on a batch.
 *   in         device, n_rows rows of n_samples samples (float, or int16_t when spec.in_dtype = MMFE_IN_S16), row r
 *              starting in_stride elements after row r - 1
 *   out        device, contiguous (n_rows, frames, feat) or (n_rows, feat, frames) per spec.layout,
 *              frames/feat as reported by mmfe_spec_out_shape (after out_frames / drop_last); elements of
 *              spec.out_dtype (float unless stated otherwise)
 *   hip_stream hipStream_t or NULL
 * Stands where the reference calls kaldi.fbank (vggsound.py:45), librosa.stft + log
 * (epic_kitchen.py:119-125), scipy.signal.stft + abs (adbox.py:20) or frame_signal. */
int mmfe_run(const mmfe_plan* plan, const void* in, int64_t in_stride, int64_t n_rows, int64_t n_samples,
             void* out, void* hip_stream);

/* mmfe_run for callers that cannot allocate device memory (code under HIP graph capture, tight serving loops, harnesses
 * that forbid hipMalloc): same arguments, same results.  No counterpart in the reference.  The one scratch buffer the
 * kernels need, the per-row maxima and minima of clamp_below_max plans, is a static device array inside the library
 * (2 x MMFE_NOALLOC_MAX_ROWS floats = 512 KiB per GPU, held until the process ends) instead of the plan's own buffer;
 * the call allocates and frees nothing.  Limits: a clamp_below_max plan takes at most MMFE_NOALLOC_MAX_ROWS rows per
 * call (more: MMFE_EINVAL, nothing is launched); every call on a GPU uses that GPU's one array, so two calls with
 * clamp_below_max plans that overlap on one GPU race (issue them on one stream).  Plans without clamp_below_max use no
 * scratch and run exactly as under mmfe_run. */
#define MMFE_NOALLOC_MAX_ROWS 65536
int mmfe_run_noalloc(const mmfe_plan* plan, const void* in, int64_t in_stride, int64_t n_rows, int64_t n_samples,
                     void* out, void* hip_stream);

/* Same transform, but row r is the slice [offsets[r], offsets[r] + n_samples) of recording
 * rec_index[r] in a packed device buffer (recording i starts rec_start[i] elements into recs).  Stands for
 * the slicing in EPICKitchen._extract_sound_feature (epic_kitchen.py:128-154) feeding _log_specgram. */
int mmfe_run_slices(const mmfe_plan* plan, const void* recs, const int64_t* rec_start, const int32_t* rec_index,
                    const int64_t* offsets, int64_t n_rows, int64_t n_samples, void* out, void* hip_stream);

/* Ragged batches in ONE launch: row r holds row_len[r] samples (device array of n_rows ints, each clamped to
 * [0, n_samples]); n_samples is the length of the longest row and fixes the output shape exactly as in mmfe_run.  Every
 * row is transformed as if it were passed alone with its own length (its own padding at its own end, its own frame
 * count); frames a shorter row does not have are filled like the frames beyond out_frames' natural count
 * ((pad_value + out_shift) * out_scale).  Stands for a DataLoader batch that mixes lengths: the reference feeds
 * interior (30 672-sample) and edge (30 696-sample) EPIC slices through the same _log_specgram
 * (epic_kitchen.py:143-154, both give 256 frames) and pads VGGSound clips of any length to 384 frames
 * (vggsound.py:48-56).  FBANK and LOGSPEC kinds without clamp_below_max.  The first win_len elements of `in` / `recs`
 * must be readable (the kernels park masked lanes there). */
int mmfe_run_ragged(const mmfe_plan* plan, const void* in, int64_t in_stride, const int32_t* row_len, int64_t n_rows,
                    int64_t n_samples, void* out, void* hip_stream);
int mmfe_run_slices_ragged(const mmfe_plan* plan, const void* recs, const int64_t* rec_start, const int32_t* rec_index,
                           const int64_t* offsets, const int32_t* row_len, int64_t n_rows, int64_t n_samples, void* out,
                           void* hip_stream);

/* Sum and sum of squares (float64) of n device floats, accumulated into sums[0], sums[1] (device,
 * caller zeroes them).  Stands for the two DataLoader passes of cal_norm (vggsound.py:85-107). */
int mmfe_feature_sums(const float* x, int64_t n, double* sums, int device, void* hip_stream);

/* Name of the kernel family that serves the plan ("fbank512", "rfft400", "dftgen", "stft32", "frame"); a static
 * string, never NULL.  Diagnostic: the reference has one code path per transform, so nothing there corresponds;
 * tests use it to make sure a parameter set reaches the kernel they mean to exercise. */
const char* mmfe_plan_kernel(const mmfe_plan* plan);

/* ---- patch embedding: the consumer's first layer --------------------------------------------------------------
 * The encoders turn the spectrogram into tokens with one 16 x 16 / stride-16 convolution, PatchEmbed.forward
 * (classification/vggsound/models/vit_model.py:193-199) with the projection AudioTransformer installs at vit_model.py:435:
 *     tokens = proj(x).flatten(2).transpose(1, 2)          x: (B, 1, H, W)  ->  (B, P, embed_dim), P = (H/16) * (W/16)
 * computed under @autocast() (vit_model.py:388) in a 16-bit type.  mmfe_patch_embed_create packs Conv2d.weight
 * ((embed_dim, 1, 16, 16) contiguous = embed_dim rows of 256 floats) and Conv2d.bias (embed_dim floats or NULL), rounded to
 * compute_dtype (MMFE_OUT_F16: what autocast uses on a GPU; MMFE_OUT_BF16), into matrix-pipe operand order on `device`;
 * the image (in_dtype MMFE_IN_F32) is rounded to compute_dtype on the way in, or already holds that type (in_dtype MMFE_IN_F16 /
 * MMFE_IN_BF16: the spectrogram as the front-end kernels store it with out_dtype float16 / bfloat16, bit-identical to the cast);
 * products are accumulated in float32, tokens are stored as out_dtype.
 * Limits: patch = 16, embed_dim 384 or 768, width a multiple of 4 (8 for 16-bit images); rows / columns beyond the last whole
 * patch are ignored, as the convolution ignores them. */
typedef struct mmfe_patch_embed mmfe_patch_embed;
int mmfe_patch_embed_create(int32_t height, int32_t width, int32_t patch, int32_t embed_dim, const float* weight, const float* bias,
                            int32_t in_dtype, int32_t compute_dtype, int32_t out_dtype, int device, mmfe_patch_embed** out_handle);
int mmfe_patch_embed_destroy(mmfe_patch_embed* handle);
/* New weights for an existing handle, read from DEVICE memory (the Conv2d parameters of a model in training, after an optimizer
 * step: vanilla_single.py:75-80): weight_dev (embed_dim, 256) float32 contiguous, bias_dev embed_dim floats or NULL (zeros).  One
 * small kernel on hip_stream re-packs and rounds them as mmfe_patch_embed_create does on the host: no allocation, no
 * synchronisation; calls of mmfe_patch_embed_run issued later on the same stream use the new weights. */
int mmfe_patch_embed_update(mmfe_patch_embed* handle, const float* weight_dev, const float* bias_dev, void* hip_stream);
/* P and embed_dim of the tokens one image yields. */
int mmfe_patch_embed_shape(const mmfe_patch_embed* handle, int64_t* n_patches, int64_t* embed_dim);
/* x: device, n_batch images (elements of in_dtype) of height x width (unit column stride, row stride = width), image b starting
 * x_batch_stride elements after image b - 1 (16-byte aligned); out: device, (n_batch, P, embed_dim) of out_dtype, image b's
 * tokens starting out_batch_stride elements after image b - 1's (so that a caller can leave room for a class token in
 * front, vit_model.py:382-383).  Asynchronous on hip_stream, allocates nothing. */
int mmfe_patch_embed_run(const mmfe_patch_embed* handle, const void* x, int64_t x_batch_stride, int64_t n_batch, void* out,
                         int64_t out_batch_stride, void* hip_stream);

/* ---- rotary positions with several axes ------------------------------------------------------------------------------
 * The tokens of mmfe_patch_embed_run sit on a grid (frequency and time of a spectrogram; height and width of an image; with a time
 * axis in front, video).  Element pair i of every query and key head turns by position[axis(i)] * theta_i.  sections[a] pairs
 * belong to axis a, in order; R = sum of the sections; the dim - 2 R elements behind them pass through.
 *   ladder   MMFE_ROTARY_SHARED: theta_i = base^(-i / R), one ladder over all pairs;  MMFE_ROTARY_PER_AXIS: base^(-j / sections[a])
 *            for the j-th pair of axis a
 *   pairing  MMFE_ROTARY_HALVES: elements (i, i + R);  MMFE_ROTARY_ADJACENT: elements (2 i, 2 i + 1)
 * Angles are formed in float64.  The reference adds a learned position table instead (classification/vggsound/models/vit_model.py:
 * 384-385); nothing there corresponds.  The handle owns the frequency table and may be shared between threads and streams. */
#define MMFE_ROTARY_SHARED    0
#define MMFE_ROTARY_PER_AXIS  1
#define MMFE_ROTARY_HALVES    0
#define MMFE_ROTARY_ADJACENT  1
typedef struct mmfe_rotary mmfe_rotary;
typedef struct mmfe_rotary_args {
    int32_t struct_size;    /* = sizeof(mmfe_rotary_args) */
    int32_t dtype;          /* MMFE_OUT_F32 / _F16 / _BF16: element type of q, k and their outputs */
    int32_t pos_64;         /* 1: positions are int64_t; 0: int32_t */
    int32_t inverse;        /* 1: rotate by the negative angle (the gradient) */
    int32_t heads_q, heads_k;
    int32_t dim;            /* elements of a head, 2 R to 1024, unit stride */
    int32_t reserved;
    int64_t n_batch, n_tokens;
    const void* q;          /* device, (n_batch, n_tokens, heads_q, dim) with strides q_stride (elements) */
    void* q_out;            /* may be q itself with the same strides: in place */
    const void* k;
    void* k_out;
    int64_t q_stride[3], q_out_stride[3], k_stride[3], k_out_stride[3];
    const void* positions;  /* device, (axes, n_batch, n_tokens) with strides pos_stride (batch stride 0: shared) */
    int64_t pos_stride[3];
} mmfe_rotary_args;
int mmfe_rotary_create(int32_t n_axes, const int32_t* sections, int32_t ladder, int32_t pairing, double base, int device, mmfe_rotary** out_handle);
int mmfe_rotary_destroy(mmfe_rotary* handle);
/* One launch for q and k; either may have no heads.  Asynchronous on hip_stream, allocates nothing. */
int mmfe_rotary_run(const mmfe_rotary* handle, const mmfe_rotary_args* args, void* hip_stream);

/* ---- attention over the encoders' tokens ------------------------------------------------------------------------------------
 * The product the encoders spend their time in (Attention.forward, classification/vggsound/models/vit_model.py:43-69, computed there as
 * two matrix products around a softmax over a materialised score tensor), over documents of different lengths:
 *     s = scale q k^T;   cap > 0: s = cap tanh(s / cap);   slopes: s -= slopes[head] |i + (len_k - len_q) - j|
 *     out = softmax(s) v over the keys j of row i's document with  not causal, or j <= i + len_k - len_q, or j < prefix[document]
 * Rows that see no key, and rows no document holds, give zeros (lse -inf).  Key head of query head h: h / (heads / kv_heads).
 *   packed = 0   n_docs batch entries of q_rows x k_rows; q_len / k_len (device, n_docs entries, clamped to [0, rows]) or NULL = all
 *   packed = 1   document d holds rows q_off[d] .. q_off[d + 1] - 1 of q_rows and keys k_off[d] .. of k_rows (device, n_docs + 1
 *                nondecreasing entries each, clamped to the rows); batch strides are ignored and must be 0
 * float16 / bfloat16, head size a multiple of 8 up to 128; strides in elements, multiples of 8, unit stride inside the heads,
 * 16-byte aligned; 2^-90 <= scale <= 2^126, cap finite.  Scores, softmax and sums are float32; the softmax's values are rounded to the 16-bit type for the product with v.
 * Values of rows outside a document never enter it; inside one, a NaN or infinity of a key that a causal mask hides may reach rows
 * up to 63 before it.  Asynchronous on hip_stream, allocates nothing. */
typedef struct mmfe_attention_args {
    int32_t struct_size;      /* = sizeof(mmfe_attention_args) */
    int32_t dtype;            /* MMFE_OUT_F16 / MMFE_OUT_BF16, of every 16-bit tensor */
    int32_t n_docs, heads, kv_heads, dim;
    int32_t packed, causal;
    float   scale, cap;
    int64_t q_rows, k_rows;
    const void *q, *k, *v;
    const int32_t *q_len, *k_len, *q_off, *k_off;
    const int32_t* prefix;    /* n_docs entries or NULL; needs causal */
    const float* slopes;      /* heads entries or NULL */
    void* out;
    void* out_rest;           /* like out (same strides): what the rounding of out lost, for the gradients; NULL: not wanted */
    float* lse;               /* (n_docs,) heads, q_rows by lse_stride; NULL: not wanted (backward needs it) */
    int64_t q_stride[3], k_stride[3], v_stride[3], out_stride[3];   /* batch, row, head */
    int64_t lse_stride[2];    /* batch, head; rows are contiguous */
} mmfe_attention_args;
/* Bytes of device memory mmfe_attention_forward needs for these arguments (the keys are cut where there are few blocks of rows, into parts
 * whose results are joined): 16-byte aligned, the call's own until it has run.  0: none.  -1: the arguments are refused. */
int64_t mmfe_attention_workspace(const mmfe_attention_args* args);
int mmfe_attention_forward(const mmfe_attention_args* args, void* workspace, int device, void* hip_stream);

/* Gradients of q, k and v from the forward call's arguments (with its out, lse and, where it was stored, out_rest) and the gradient of out.  Those of a shared key
 * head are summed over its query heads; rows outside the documents get zeros.  Sums have a fixed order: the same call gives the
 * same bits.  lse must be the dense (n_docs,) heads, q_rows array of the forward call. */
typedef struct mmfe_attention_grads {
    int32_t struct_size;      /* = sizeof(mmfe_attention_grads) */
    int32_t reserved;
    const void* grad_out;
    void *grad_q, *grad_k, *grad_v;
    int64_t grad_out_stride[3], grad_q_stride[3], grad_k_stride[3], grad_v_stride[3];
} mmfe_attention_grads;
/* Bytes of the workspace mmfe_attention_backward needs (as mmfe_attention_workspace).  0: none, and neither out nor out_rest is read
 * (documents of up to 256 rows and keys, a key head per query head, head size up to 64). */
int64_t mmfe_attention_backward_workspace(const mmfe_attention_args* args);
int mmfe_attention_backward(const mmfe_attention_args* args, const mmfe_attention_grads* grads, void* workspace, int device, void* hip_stream);

/* ---- global norm of many tensors, and clipping by it ------------------------------------------------------------------
 * What a training step of the encoders does between backward and the optimizer (the reference's loops call the optimizer directly,
 * classification/vggsound/vanilla_single.py:75-80).  norm = (sum of all squares)^(1/2) (MMFE_NORM_2) or the largest magnitude
 * (MMFE_NORM_MAX) over all tensors, summed in float64 in a fixed order; with out != NULL every tensor times
 * min(1, max_norm / (norm + 1e-6)) goes to out[i], as out_dtype[i]; out[i] may be x[i] with the same type (in place: nothing is
 * written when the factor is 1).  A NaN norm makes every output NaN, and so does an infinite one under an infinite
 * max_norm; an infinite norm under a finite max_norm makes finite values zero.
 *   x, numel, dtype, out, out_dtype   HOST arrays of n_tensors entries, read before the call returns; x[i] / out[i] are device
 *                                     pointers of numel[i] contiguous elements (MMFE_OUT_* types), aligned to their elements
 *   partials                          device, mmfe_grad_partials(n_tensors) doubles, the call's own until it has run
 *   norm                              device, one float
 * What is written must not overlap any other tensor of the call (MMFE_EINVAL).  Asynchronous on hip_stream, allocates nothing on
 * the device. */
#define MMFE_NORM_2    2
#define MMFE_NORM_MAX  0
int64_t mmfe_grad_partials(int64_t n_tensors);
int mmfe_grad_clip(int64_t n_tensors, const void* const* x, const int64_t* numel, const int32_t* dtype, void* const* out, const int32_t* out_dtype,
                   int32_t norm_kind, float max_norm, double* partials, float* norm, int device, void* hip_stream);

#ifdef __cplusplus
}
#endif
#endif /* MMFE_H */
