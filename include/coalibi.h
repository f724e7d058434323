/*
 * coalibi.h -- C ABI of the sm_100a (B200) Co-ALiBi attention library
 * (libcoalibi_sm100.so).
 *
 * Co-ALiBi attention, per batch b, query head h, query row i and key j:
 *   p_ij = sm_scale * q_i . k_j          (masked where causal and j > i)
 *   s_ij = sigmoid(p_ij), z_ij = sum_{t >= j} s_it
 *   o_i  = softmax_j(p_ij - slope_h * z_ij) @ V
 *
 * All tensors are device pointers to contiguous row-major arrays:
 *   q, o, dout, dq     [B, Hq,  Sq,  D]
 *   k, v, dk, dv       [B, Hkv, Skv, D]      (Hq % Hkv == 0; q head h reads kv head h / (Hq/Hkv))
 *   lse, rowsig        [B, Hq,  Sq]  float32
 *   slopes             [Hq]          float32, float16 or bfloat16 (slopes_dtype)
 * with D in {64, 128}, dtype float16 or bfloat16, every pointer 16-byte aligned.
 *
 * The library never allocates device memory, never synchronises and only
 * enqueues work on the stream it is given (a cudaStream_t passed as void*; NULL
 * means the legacy default stream), which must belong to the device that holds
 * the tensors (else COALIBI_ERR_DEVICE).  Each call makes that device current
 * while it runs and puts the calling thread's previous CUDA context (possibly
 * none) back before it returns.  Calls are reentrant and thread-safe across
 * streams and devices.  Each function returns COALIBI_OK or an error code;
 * coalibi_strerror() names it.  Kernel-side failures (a bounded wait that timed
 * out) are reported asynchronously through the optional device status word.
 *
 * The forward and backward kernels are launched with programmatic stream
 * serialization: one may start its set-up while the kernel before it on the
 * stream is still finishing, but it waits for that kernel to complete before
 * it touches global memory, so stream order holds for every read and write.
 */
#ifndef COALIBI_H_
#define COALIBI_H_

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

#define COALIBI_ABI_VERSION 1

enum coalibi_dtype {
  COALIBI_F16 = 0,
  COALIBI_BF16 = 1,
  COALIBI_F32 = 2, /* only valid for slopes_dtype and weight_dtype */
  COALIBI_E4M3 = 3 /* the codes of an 8-bit cache; no argument takes it */
};

enum coalibi_error {
  COALIBI_OK = 0,
  COALIBI_ERR_NULL_POINTER = 1,
  COALIBI_ERR_HEAD_DIM = 2,     /* D not in {64, 128} */
  COALIBI_ERR_DTYPE = 3,        /* dtype not float16 / bfloat16 */
  COALIBI_ERR_SHAPE = 4,        /* non-positive sizes, Hq % Hkv != 0, or too large */
  COALIBI_ERR_ALIGNMENT = 5,    /* a pointer is not 16-byte aligned */
  COALIBI_ERR_LAUNCH = 6,       /* CUDA launch / attribute error */
  COALIBI_ERR_TENSOR_MAP = 7,   /* cuTensorMapEncodeTiled failed or unavailable */
  COALIBI_ERR_WORKSPACE = 8,    /* workspace missing or smaller than coalibi_bwd_workspace_bytes() */
  COALIBI_ERR_DEVICE = 9,       /* device is not sm_100, or the stream is on another device */
  COALIBI_ERR_TIMEOUT = 10,     /* device status only: a bounded wait expired */
  COALIBI_ERR_PAGE = 11         /* device status only: a token outside its page table, a page outside the
                                   pool, or a position outside the rotary table; the access was skipped */
};

/* Forward.  Replaces the Triton launch in co_alibi_attn/co_alibi_attn.py:44-57
 * (CoALIBIAttention.forward) and the kernel co_alibi_attn/co_alibi_fwd_kernel.py:29-127.
 * Writes o, lse = m + log(l + 1e-9) (natural log) and rowsig = sum_j sigmoid(p_ij),
 * the two float32 side outputs the backward consumes. */
typedef struct CoalibiFwdArgs {
  const void* q;
  const void* k;
  const void* v;
  const void* slopes;
  void* o;
  float* lse;
  float* rowsig;
  int B, Hq, Hkv, Sq, Skv, D;
  int dtype;        /* enum coalibi_dtype of q, k, v, o */
  int slopes_dtype; /* enum coalibi_dtype of slopes */
  int causal;       /* nonzero: top-left aligned causal mask (key j > query i masked) */
  float sm_scale;
  int* status;      /* optional device int; a kernel-side error code is CAS'ed in */
  unsigned int timeout_ms; /* bound on every in-kernel wait; 0 = default (2000 ms) */
} CoalibiFwdArgs;

int coalibi_fwd(const CoalibiFwdArgs* args, void* stream);

/* Forward for few query rows (Sq <= COALIBI_DECODE_MAX_SQ, e.g. one new token
 * against a long key/value sequence): the same arguments, mask semantics and
 * results (o, lse, rowsig) as coalibi_fwd, for the shapes the reference forward
 * launches with a nearly empty query block (co_alibi_attn/co_alibi_attn.py:44-57).
 * The keys are split into chunks (one per warp of the partial kernel) and merged
 * exactly: the sigmoid totals of the chunks to the right shift each chunk's
 * logits.  workspace: device scratch of at least coalibi_fwd_decode_workspace_bytes()
 * bytes, 16-byte aligned; contents on entry do not matter.  Sq above the limit
 * returns COALIBI_ERR_SHAPE. */
#define COALIBI_DECODE_MAX_SQ 16
size_t coalibi_fwd_decode_workspace_bytes(int B, int Hq, int Hkv, int Sq, int Skv, int D);
int coalibi_fwd_decode(const CoalibiFwdArgs* args, void* workspace, size_t workspace_bytes, void* stream);

/* Backward.  Replaces co_alibi_attn/co_alibi_attn.py:73-135 (CoALIBIAttention.backward,
 * including the dk/dv partial-buffer reduction at :132-133 and, for GQA, the group
 * sum autograd performs through repeat_interleave at :145-146) and the kernel
 * co_alibi_attn/co_alibi_bwd_kernel.py:19-146.  dk and dv have Hkv heads.
 * workspace: device scratch, 256-byte aligned, its contents on entry irrelevant.
 * The size picks the algorithm: with at least the "stored" size (what
 * coalibi_bwd_workspace_size() returns while that stays below 24 GiB) the first
 * kernel also writes P and dS as 16-bit 128 x 128 tiles -- 4 bytes per visible
 * score, 4.3 GB at B8 H16 S4096 causal, half the reference's dk/dv partial
 * buffers -- and dK, dV come from a streaming GEMM over them; with less, down to
 * coalibi_bwd_workspace_min_bytes() (8 bytes per row per 32 keys), the second
 * kernel recomputes P and dS instead.  Both agree with the reference within the
 * same tolerances; less than the minimum returns COALIBI_ERR_WORKSPACE. */
typedef struct CoalibiBwdArgs {
  const void* q;
  const void* k;
  const void* v;
  const void* o;
  const void* dout;
  const float* lse;
  const float* rowsig;
  const void* slopes;
  void* dq;
  void* dk;
  void* dv;
  void* workspace;
  size_t workspace_bytes;
  int B, Hq, Hkv, Sq, Skv, D;
  int dtype;
  int slopes_dtype;
  int causal;
  float sm_scale;
  int* status;
  unsigned int timeout_ms;
} CoalibiBwdArgs;

/* Workspace size to allocate for this call's problem and mask (args->B, Hq, Hkv,
 * Sq, Skv, D, causal; the pointers are not read): the stored layout while its
 * P / dS scratch stays below 24 GiB, else the recompute layout. */
size_t coalibi_bwd_workspace_size(const CoalibiBwdArgs* args);

/* A size that serves either mask of the problem (the larger of the two
 * coalibi_bwd_workspace_size values). */
size_t coalibi_bwd_workspace_bytes(int B, int Hq, int Hkv, int Sq, int Skv, int D);

/* The smallest workspace coalibi_bwd accepts for the problem (the recompute layout). */
size_t coalibi_bwd_workspace_min_bytes(int B, int Hq, int Hkv, int Sq, int Skv, int D);

int coalibi_bwd(const CoalibiBwdArgs* args, void* stream);

/* Backward of one key shard of longer rows (sequence / context parallelism, which
 * the reference does not have): the keys of this call are a contiguous piece of
 * each row's keys.  Same arguments as coalibi_bwd, read this way: o, lse and dout
 * are those of the whole row (so delta and P are global); rowsig is the sigmoid
 * total of this call's keys plus that of every key right of them; dA_carry_in
 * [B * Hq * Sq] float32 is sum_t P_it (dP_it - delta_i) over the keys left of them.
 * dq, dk and dv are this shard pair's contributions (sum them over the shards). */
int coalibi_bwd_carry(const CoalibiBwdArgs* args, const float* dA_carry_in, void* stream);

/* Profiling aid with no counterpart in the reference: launch only the backward
 * kernels selected by phase_mask (bit 0: delta = rowsum(dO * O) pre-pass, bit 1:
 * pass A -> dq and, in the workspace, P / dS tiles or the per-32-key carries,
 * bit 2: pass B -> dk, dv).
 * Phases read what earlier phases wrote into the workspace, so they must run in
 * order on one stream; coalibi_bwd(args, s) == coalibi_bwd_phases(args, 7, s). */
int coalibi_bwd_phases(const CoalibiBwdArgs* args, int phase_mask, void* stream);

/* Size of the static device scratch used by coalibi_bwd_noalloc (64 MiB). */
#define COALIBI_NOALLOC_SCRATCH_BYTES ((size_t)64 << 20)

/* Backward that allocates nothing and needs no workspace: same arguments and
 * results as coalibi_bwd, with args->workspace / workspace_bytes ignored.  It has
 * no counterpart in the reference.  It is for callers that cannot allocate device
 * memory at the call -- a plugin host or FFI caller that owns only the tensors
 * it passes, or code that must avoid cudaMalloc there because it can synchronise
 * the device.  Its scratch is one file-scope device array of
 * COALIBI_NOALLOC_SCRATCH_BYTES per GPU, held until the process exits; the
 * backward runs the stored path when its scratch fits there, else the recompute
 * path; problems needing more (coalibi_bwd_workspace_min_bytes() > that) return
 * COALIBI_ERR_WORKSPACE without launching.  The first call on each device looks up the array's device
 * address (cudaGetSymbolAddress); make it before any stream capture.  The address
 * is not looked up again, so it is stale after cudaDeviceReset on that device.
 * All calls on a device share the array, so calls that overlap on the GPU race:
 * serialise them. */
int coalibi_bwd_noalloc(const CoalibiBwdArgs* args, void* stream);

/* Self-test of the kernels' bounded waits, with no counterpart in the reference:
 * enqueues one CTA whose warps wait on mbarriers that nothing ever arrives on.
 * Every such wait in this library gives up after its timeout, raises the CTA's
 * abort flag and records COALIBI_ERR_TIMEOUT in the device word *status (if it
 * still holds 0), so the kernel ends after about timeout_ms (0: the default of
 * 2000) and the CUDA context stays usable.  Returns the launch result; read
 * *status after synchronising the stream. */
int coalibi_selftest_wait_timeout(unsigned int timeout_ms, int* status, void* stream);

/* The launch configuration this library picks for a problem, as one line of
 * text: the counterpart of the reference's COALIBI_VERBOSE=1 print of the
 * configuration its autotuner chose (co_alibi_attn/co_alibi_attn.py:58-63 for the
 * forward, :125-130 for the backward).  which: 0 forward (coalibi_fwd), 1 decode
 * forward (coalibi_fwd_decode), 2 backward (coalibi_bwd, with the workspace of
 * coalibi_bwd_workspace_size); causal: the mask; device: the CUDA device index (for
 * its SM count).  Writes a NUL-terminated description into buf, truncated to
 * buf_len bytes.  Launches nothing and changes no CUDA state. */
int coalibi_describe_launch(int which, int B, int Hq, int Hkv, int Sq, int Skv, int D, int causal, int device,
                            char* buf, size_t buf_len);

/* ---------------------------------------------------------------------------
 * Serving: a decoding step of a Co-ALiBi model over a paged key/value cache.
 * The reference has no counterpart of these.
 *
 * A cache is a pool of pages: k_pages and v_pages hold n_pages pages of page_size
 * tokens (a multiple of 16) for each of Hkv heads, element (page, head, slot, d) at
 * page * stride[0] + head * stride[1] + slot * stride[2] + d; strides in elements,
 * multiples of 8, bases 16-byte aligned.  Token t of request b lives in page
 * page_table[b * table_stride + t / page_size], slot t % page_size.  Lengths and
 * tables are read on the device, so a captured graph can replay as they change;
 * entries past a request's tokens are never used.  A token outside the table or a
 * page outside the pool is skipped and reported as COALIBI_ERR_PAGE in *status; a token
 * whose position has no row in the rotary table is appended unrotated and reported too.
 * ------------------------------------------------------------------------- */

/* Append the S new tokens (count[b] of them when count is given) of each request at
 * tokens start[b], start[b] + 1, ... of its cache.  With rot > 0 the first rot
 * elements of each key, and of each query when q is given, are rotated by the angle
 * of the token's position (positions[b, i], default start[b] + i): pairs
 * (x[i], x[i + rot / 2]), or (x[2i], x[2i + 1]) when interleaved, become
 * (a cos - b sin, b cos + a sin) in float32, rounded once.  q_out rows past count[b]
 * are zero.  Strides of k, v, q, q_out: batch, head, token; multiples of 8. */
typedef struct CoalibiPagedAppendArgs {
  const void* k;
  const void* v;
  const void* q;          /* optional: queries to rotate */
  void* q_out;
  void* k_pages;
  void* v_pages;
  const int* page_table;  /* [B, max_pages] */
  const int* start;       /* [B] */
  const int* count;       /* [B]; NULL: S */
  const int* positions;   /* [B, S] contiguous; NULL: start[b] + i */
  const float* cos;       /* [n_pos, rot / 2]; NULL with rot = 0 */
  const float* sin;
  int* status;            /* optional device int */
  long long k_stride[3], v_stride[3], q_stride[3], q_out_stride[3];
  long long k_page_stride[3], v_page_stride[3]; /* page, head, slot */
  long long table_stride;
  int B, Hq, Hkv, S, D;   /* Hq read only with q */
  int page_size, max_pages, n_pages;
  int rot, n_pos, interleaved; /* rot: a multiple of 16, at most D */
  int dtype;
} CoalibiPagedAppendArgs;

int coalibi_paged_append(const CoalibiPagedAppendArgs* args, void* stream);

/* Co-ALiBi attention of Sq query rows per request over its paged cache: the
 * ctx_lens[b] context tokens, which every row sees, and the up to Sq drafted tokens
 * after them, of which row i sees token ctx_lens[b] + t where bit t of
 * tree_mask[b * mask_stride + i] is set (tree_mask NULL: bits 0 .. i, a chain; Sq = 1
 * is one decoding step).  z sums the sigmoids of the keys the row sees, in cache order;
 * a row that sees nothing gives 0.  Drafted tokens that no row of a request sees are
 * not read.  workspace: coalibi_paged_attention_workspace_bytes() bytes, 16-byte
 * aligned, contents on entry irrelevant, not shared by calls that may overlap. */
#define COALIBI_TREE_MAX_SQ 64
typedef struct CoalibiPagedAttentionArgs {
  const void* q;          /* [B, Hq, Sq, D] by stride */
  void* o;
  const void* k_pages;
  const void* v_pages;
  const void* slopes;     /* [Hq], slopes_dtype */
  const int* page_table;
  const int* ctx_lens;    /* [B] */
  const long long* tree_mask;
  int* status;
  long long q_stride[3], o_stride[3]; /* batch, head, row; multiples of 8 */
  long long k_page_stride[3], v_page_stride[3];
  long long table_stride, mask_stride; /* mask_stride 0: one mask for all requests */
  int B, Hq, Hkv, Sq, D;
  int page_size, max_pages, n_pages;
  int dtype, slopes_dtype;
  float sm_scale;
} CoalibiPagedAttentionArgs;

size_t coalibi_paged_attention_workspace_bytes(int B, int Hq, int Hkv, int Sq, int D);
int coalibi_paged_attention(const CoalibiPagedAttentionArgs* args, void* workspace, size_t workspace_bytes,
                            void* stream);

/* The same cache in 8 bits.  k_pages and v_pages hold e4m3 codes (strides multiples of 16), and each
 * block of 16 tokens of a page and head has a float32 scale at page * stride[0] + head * stride[1] + slot / 16: a
 * value is its code times the scale of its block.  The append writes powers of two; reading and attention take
 * any finite scale. */
#define COALIBI_QUANT_BLOCK 16
typedef struct CoalibiCacheScales {
  float* k; /* [n_pages, Hkv, page_size / 16] */
  float* v;
  long long k_stride[2], v_stride[2]; /* page, head */
} CoalibiCacheScales;

/* coalibi_paged_append into such a cache.  A block that the new tokens begin takes the least power of
 * two, and at least 2^-100, by which its largest finite value is at most 448; one that held tokens before
 * them keeps its scale unless that is smaller, and if not its old codes move to the new scale.  Values are
 * rounded once, rotated keys from float32; infinities become NaN. */
int coalibi_paged_append8(const CoalibiPagedAppendArgs* args, const CoalibiCacheScales* scales, void* stream);

/* coalibi_paged_attention over such a cache; the workspace is that of
 * coalibi_paged_attention8_workspace_bytes(). */
size_t coalibi_paged_attention8_workspace_bytes(int B, int Hq, int Hkv, int Sq, int D);
int coalibi_paged_attention8(const CoalibiPagedAttentionArgs* args, const CoalibiCacheScales* scales, void* workspace,
                             size_t workspace_bytes, void* stream);

/* Tokens of such a cache in 16 bits: token positions[b, i] of request b becomes row i of k and v.
 * Rows of a negative position are zero, and so are those outside the table or the pool, which are
 * reported.  Values are rounded once; one past the type's largest is that. */
typedef struct CoalibiPagedReadArgs {
  const void* k_pages;
  const void* v_pages;
  const int* page_table;  /* [B, max_pages] */
  const int* positions;   /* [B, S] contiguous */
  void* k;                /* [B, Hkv, S, D] contiguous, dtype; 32-byte aligned */
  void* v;
  int* status;
  long long k_page_stride[3], v_page_stride[3]; /* page, head, slot */
  long long table_stride;
  int B, Hkv, S, D;
  int page_size, max_pages, n_pages;
  int dtype;
} CoalibiPagedReadArgs;

int coalibi_paged_read8(const CoalibiPagedReadArgs* args, const CoalibiCacheScales* scales, void* stream);

/* Heads of a fused projection.  qkv [B, S, Hq + 2 Hkv, D]: query, key and value heads of each token.
 * Forward: q [B, Hq, S, D], k and v [B, Hkv, S, D] by stride; with x a row of a query or key head,
 *   y = R(x / sqrt(mean(x^2) + eps) * weight),
 * R the rotation of coalibi_paged_append by the angles of position positions[b, i], else start[b] + i,
 * else i (rot = 0: none; a position outside the table leaves the row unrotated and is reported as
 * COALIBI_ERR_PAGE); values are moved.  Arithmetic is float32, rounded once.
 * Backward: q, k and v are the gradients of the three (read); dqkv [B, S, Hq + 2 Hkv, D] contiguous, and
 * dq_weight, dk_weight [D] (weight_dtype; NULL: not wanted) are written.  Sums are float32, in a fixed
 * order: results repeat bit for bit.  workspace: coalibi_heads_bwd_workspace_bytes(), 16-byte aligned,
 * contents on entry irrelevant, not shared by calls that may overlap. */
typedef struct CoalibiHeadsArgs {
  const void* qkv;
  void* q;
  void* k;
  void* v;
  const void* q_weight;  /* [D]; NULL: ones */
  const void* k_weight;
  const float* cos;      /* [n_pos, rot / 2]; NULL with rot = 0 */
  const float* sin;
  const int* start;      /* [B]; NULL: 0 */
  const int* positions;  /* [B, S] contiguous; NULL: start[b] + i */
  int* status;           /* optional device int */
  void* dqkv;
  void* dq_weight;
  void* dk_weight;
  long long qkv_stride[3];                        /* batch, token, head; multiples of 8 */
  long long q_stride[3], k_stride[3], v_stride[3]; /* batch, head, token; multiples of 8 */
  int B, S, Hq, Hkv, D;
  int rot, n_pos, interleaved; /* rot: a multiple of 16, at most D */
  int dtype, weight_dtype;     /* weight_dtype: dtype or COALIBI_F32 */
  float eps;
} CoalibiHeadsArgs;

int coalibi_heads_fwd(const CoalibiHeadsArgs* args, void* stream);
size_t coalibi_heads_bwd_workspace_bytes(int Hq, int Hkv, int D);
int coalibi_heads_bwd(const CoalibiHeadsArgs* args, void* workspace, size_t workspace_bytes, void* stream);

/* Draw one token for each row of logits.  Tokens are ranked by (logit descending,
 * index ascending) and weighted w = exp((logit - max) / temperature); kept are the
 * first top_k (0: all), of those the shortest prefix whose weights reach top_p of
 * their sum (>= 1: all, at least one stays), of those w >= min_p.  The token is the
 * kept one with the largest w / noise: with noise drawn from Exp(1) that samples the
 * renormalised distribution.  temperature <= 0: the first of the ranking.  Logits of
 * -inf or NaN are never drawn; +inf logits share all the weight.  logprobs[b] is the
 * drawn token's log-probability among the kept.  A row with nothing to draw gives
 * token -1, logprob -inf.  The masses that top_p cuts are 64-bit fixed point (weights
 * in units of 2^-31, so that the order of atomics does not matter); the sum behind logprobs
 * adds float32 weights, in double across chunks and in a fixed order.  Results repeat bit for
 * bit. */
#define COALIBI_SAMPLE_MAX_VOCAB (1 << 21)
typedef struct CoalibiSampleArgs {
  const void* logits;       /* [B, V], row stride logits_stride elements */
  const float* noise;       /* [B, V], row stride noise_stride */
  const float* temperature; /* [B], or NULL: temperature_all; the same for the next three */
  const int* top_k;
  const float* top_p;
  const float* min_p;
  long long* tokens;        /* [B] */
  float* logprobs;          /* [B] */
  long long logits_stride, noise_stride;
  int B, V;
  int dtype;                /* float16, bfloat16 or float32 */
  float temperature_all;
  int top_k_all;
  float top_p_all, min_p_all;
} CoalibiSampleArgs;

int coalibi_sample(const CoalibiSampleArgs* args, void* stream);

/* Static name of an error code. */
const char* coalibi_strerror(int code);

/* COALIBI_ABI_VERSION of the loaded library. */
int coalibi_abi_version(void);

/* Detail (driver/runtime result and arguments) of the last failing call made by
 * the calling thread; "" if none.  No counterpart in the reference. */
const char* coalibi_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* COALIBI_H_ */
