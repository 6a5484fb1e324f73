/*
 * srs_b200.h — C ABI of the sm_100a stochastic-rounding optimizer library.
 *
 * Every entry point takes plain device addresses, element counts, POD
 * scalars and a cudaStream_t passed as `void*`.  Nothing here allocates
 * device memory: callers own every buffer (inputs, outputs and the row
 * tables of the multi-tensor steps).  Work is enqueued on the given stream
 * of the calling thread's current device; no entry point synchronises
 * (srs_product_status apart).
 *
 * Return value: SRS_OK (0) or a negative SRS_ERR_* code.  The text of the
 * most recent failure on the calling thread is available from
 * srs_last_error().  No entry point aborts the process.
 *
 * Counter-hash RNG contract (identical to the Python `sr_states` package):
 *   h32(x)        x ^= x>>16; x *= 0x7FEB352D; x ^= x>>15; x *= 0x846CA68B; x ^= x>>16   (mod 2^32)
 *   update_key    k = h32(seed_lo ^ 0x9E3779B9); k = h32(k ^ seed_hi); k = h32(k ^ step_lo);
 *                 k = h32(k ^ step_hi); k = h32(k ^ param_index)
 *   state_key     h32(update_key ^ state_index)
 *   element e of a stored state uses h32((e + offset + state_key) mod 2^32);
 *   element e of a standalone cast uses h32((e + offset + seed) mod 2^32).
 */
#ifndef SRS_B200_H
#define SRS_B200_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SRS_ABI_VERSION 6

/* ---- status codes ------------------------------------------------------ */
#define SRS_OK 0
#define SRS_ERR_INVALID_ARGUMENT (-1) /* bad pointer, size, format, rule or flag */
#define SRS_ERR_UNSUPPORTED_DEVICE (-2) /* current device is not compute capability 10.0 */
#define SRS_ERR_CUDA (-3)             /* a CUDA runtime call failed (launch, attribute query) */
#define SRS_ERR_WAIT (-4)             /* a wait in an earlier product kernel ran out */

/* ---- storage formats (state, cast output) ------------------------------ */
#define SRS_FMT_F32 0
#define SRS_FMT_BF16 1
#define SRS_FMT_F16 2
#define SRS_FMT_E4M3 3 /* torch.float8_e4m3fn, saturating to +-448 */
#define SRS_FMT_E5M2 4 /* torch.float8_e5m2, saturating to +-57344 */

/* ---- rounding rules ---------------------------------------------------- */
#define SRS_RULE_NEAREST 0    /* round to nearest, ties to even */
#define SRS_RULE_STOCHASTIC 1 /* counter-hash stochastic rounding */
/* Round toward zero: the format's value of largest magnitude not above |x|,
 * sign kept (BF16: the high half of the FP32 encoding).  Finite values never
 * become infinite; +-Inf stays infinite in BF16/FP16 and saturates in FP8; NaN
 * is stored as under the other rules.  Not a reference built-in: it is the
 * native implementation a custom rule registered through
 * register_rounding(..., native="toward_zero") runs (the reference's custom
 * rules, sr_states/rounding.py:28-66, run as Triton callbacks). */
#define SRS_RULE_TOWARD_ZERO 2

/* ---- multi-tensor row table -------------------------------------------- */
#define SRS_ROW_PARAM_BF16 0x1u  /* parameter is BF16 (else FP32) */
#define SRS_ROW_GRAD_BF16 0x2u   /* gradient is BF16 (else FP32) */
#define SRS_ROW_VECTOR_OK 0x4u   /* every base address is aligned for 8-element vector access */
#define SRS_ROW_CLASS_SHIFT 8    /* bits 8..15: index of the row's AdamW step class */
#define SRS_MAX_STEP_CLASSES 32
/* `uniform_kind` of the multi-tensor steps: the (SRS_ROW_PARAM_BF16 |
 * SRS_ROW_GRAD_BF16) bits every row shares, or SRS_KIND_MIXED.  It selects a
 * kernel specialised for that dtype pair; rows that do not match it still run
 * correctly on a generic path. */
#define SRS_KIND_MIXED 0xFFFFFFFFu

/*
 * One row = one contiguous run of `numel` elements of one parameter (a whole
 * parameter, or its intersection with this rank's ZeRO-1 shard).  Rows are
 * ordered by tile_begin; row i covers tiles [tile_begin_i, tile_begin_{i+1})
 * and tile_begin_i + ceil(numel_i / srs_tile_elems()) == tile_begin_{i+1}.
 */
typedef struct srs_row {
  uint64_t param;       /* device address of the parameter run (FP32 or BF16)    */
  uint64_t grad;        /* device address of the gradient run (FP32 or BF16)     */
  uint64_t state[2];    /* device addresses of the state runs (state[1]: AdamW)  */
  int64_t numel;        /* > 0                                                    */
  int64_t tile_begin;   /* first tile of this row in the launch's tile space      */
  uint32_t param_index; /* global parameter position (low 32 bits), or the update
                           key itself when the launch uses SRS_KEY_GIVEN          */
  uint32_t offset;      /* flat element index of element 0 within its parameter,
                           mod 2^32 (the shard start of the RNG contract)        */
  uint32_t flags;       /* SRS_ROW_* bits and the step class                     */
  uint32_t reserved;    /* zero                                                   */
} srs_row;

/* How the per-row update key is obtained. */
#define SRS_KEY_DERIVE 0 /* update_key(seed words, step words, row.param_index) */
#define SRS_KEY_GIVEN 1  /* row.param_index already holds the update key        */

typedef struct srs_rng {
  uint32_t seed_lo, seed_hi; /* low 64 bits of the group seed   */
  uint32_t step_lo, step_hi; /* low 64 bits of the global RNG step */
  int32_t key_mode;          /* SRS_KEY_DERIVE or SRS_KEY_GIVEN  */
} srs_rng;

/*
 * AdamW scalars, each the FP32 rounding of the double-precision expression:
 *   beta1, beta2, one_minus_beta1 = 1-beta1, one_minus_beta2 = 1-beta2,
 *   eps, decay = 1 - lr*weight_decay,
 *   per step class c (bias-correction step t_c):
 *     neg_step_size[c] = -lr / (1 - beta1^t_c),  bias2_sqrt[c] = (1 - beta2^t_c)^0.5
 * Per element (FP32, each operation rounded once):
 *   m' = fma(g, 1-b1, m*b1);  v' = fma((1-b2)*g, g, v*b2)
 *   d  = sqrt(v') / bias2_sqrt + eps;  p' = p*decay + (neg_step_size*m') / d
 */
typedef struct srs_adamw_hparams {
  float beta1, beta2, one_minus_beta1, one_minus_beta2;
  float eps, decay;
  int32_t n_step_classes; /* 1..SRS_MAX_STEP_CLASSES */
  float neg_step_size[SRS_MAX_STEP_CLASSES];
  float bias2_sqrt[SRS_MAX_STEP_CLASSES];
} srs_adamw_hparams;

/* SGDM scalars: u' = u*momentum + g;  p' = fma(u', neg_lr, p), neg_lr = -lr. */
typedef struct srs_sgdm_hparams {
  float momentum;
  float neg_lr;
} srs_sgdm_hparams;

/* ---- library information ----------------------------------------------- */
int srs_abi_version(void);
/* Elements per tile of the multi-tensor steps (row tile_begin arithmetic). */
int64_t srs_tile_elems(void);
/* Text of the last failure on this thread ("" if none). */
const char* srs_last_error(void);
/* SRS_OK if the current device can run the kernels (compute capability 10.0). */
int srs_check_device(void);

/* ---- standalone cast ---------------------------------------------------
 * Replaces sr_states/triton/cast.py:32-60 (`cast`) and
 * sr_states/triton/sr_cast.py:89-128 (`sr_cast_bf16`, `rn_cast_bf16`).
 * y[e] = round(x[e]) into `out_format` under `rule`; the stochastic counter of
 * element e is (e + offset + seed) mod 2^32.  SRS_FMT_F32 copies.  x and y must
 * not overlap.  n == 0 is a no-op.
 */
int srs_cast(const float* x, void* y, int64_t n, int out_format, int rule, uint32_t seed,
             uint32_t offset, int grid_ctas, void* stream);

/* ---- fused multi-tensor steps -------------------------------------------
 * Replace the per-bucket launches of sr_states/triton/adamw.py:303-317
 * (_multi_adamw_kernel) and sr_states/triton/sgd.py:214-237
 * (_multi_sgdm_kernel): ONE launch covers every row of a parameter group on
 * one device, whatever the rows' parameter/gradient dtypes and AdamW
 * bias-correction steps.  `rows` is a device array of n_rows srs_row;
 * n_tiles = tile_begin of the last row + its tile count.  grid_ctas <= 0
 * selects the persistent grid (a multiple of the SM count).
 */
int srs_adamw_multi(const srs_row* rows, int64_t n_rows, int64_t n_tiles, int m_format,
                    int m_rule, int v_format, int v_rule, const srs_adamw_hparams* hp,
                    const srs_rng* rng, uint32_t uniform_kind, int grid_ctas, void* stream);

int srs_sgdm_multi(const srs_row* rows, int64_t n_rows, int64_t n_tiles, int u_format,
                   int u_rule, const srs_sgdm_hparams* hp, const srs_rng* rng,
                   uint32_t uniform_kind, int grid_ctas, void* stream);

/* ---- fused step + all-gather over peer memory ----------------------------
 * No counterpart in the reference (it has no sharded step; this is the
 * ZeRO-1 all-gather of the updated parameters fused into the step).  With
 * every rank's parameters in a flat buffer of identical layout, the step
 * stores each updated parameter vector both locally and at the same offset of
 * every peer's buffer (plain stores through NVLink peer mappings), so no
 * separate all-gather runs.  delta_*[w] = (peer w's buffer) - (this rank's
 * buffer) in this process's address space, for FP32 and BF16 parameters.
 * The caller orders the step against the peers (a barrier before, so no peer
 * still reads its replica, and one after, before anyone uses the result).
 */
#define SRS_MAX_PEERS 7
/* How the updated parameters reach the replicas (srs_peers.mode):
 *   SRS_PEERS_STORE      each vector is stored locally and at delta_*[w] for
 *                        every peer w (plain stores through peer mappings);
 *   SRS_PEERS_MULTICAST  the caller's flat buffers are bound to an NVLink
 *                        multicast object spanning every rank (this one
 *                        included) and mc_delta_* = (multicast address of the
 *                        buffer) - (this rank's buffer): each aligned 8-element
 *                        vector is written ONCE, with multimem.st, and NVSwitch
 *                        delivers it to every replica, the local one included.
 *                        Elements outside aligned vectors (row tails, rows
 *                        without SRS_ROW_VECTOR_OK), which multimem cannot
 *                        store at 2-byte granularity, take the SRS_PEERS_STORE
 *                        path, so delta_*[] must hold the peers as well.
 * Both end with a system-scope fence (and a proxy fence for the multicast
 * alias), so the caller's barrier after the step publishes every replica. */
#define SRS_PEERS_STORE 0
#define SRS_PEERS_MULTICAST 1
typedef struct srs_peers {
  int32_t n_peers; /* 0..SRS_MAX_PEERS */
  int32_t mode;    /* SRS_PEERS_STORE or SRS_PEERS_MULTICAST */
  int64_t delta_f32[SRS_MAX_PEERS];
  int64_t delta_bf16[SRS_MAX_PEERS];
  int64_t mc_delta_f32;  /* SRS_PEERS_MULTICAST: multicast address - local buffer */
  int64_t mc_delta_bf16;
} srs_peers;

int srs_adamw_multi_gather(const srs_row* rows, int64_t n_rows, int64_t n_tiles, int m_format,
                           int m_rule, int v_format, int v_rule, const srs_adamw_hparams* hp,
                           const srs_rng* rng, uint32_t uniform_kind, const srs_peers* peers,
                           int grid_ctas, void* stream);

int srs_sgdm_multi_gather(const srs_row* rows, int64_t n_rows, int64_t n_tiles, int u_format,
                          int u_rule, const srs_sgdm_hparams* hp, const srs_rng* rng,
                          uint32_t uniform_kind, const srs_peers* peers, int grid_ctas,
                          void* stream);

/* ---- tile ranges and copies for a pipelined exchange ---------------------
 * No counterpart in the reference.  The same steps over the tiles
 * [tile_lo, tile_hi) of the table only (0 <= tile_lo <= tile_hi <= n_tiles):
 * a sharded step split into chunks, each chunk's updated parameters sent to
 * the peers by srs_copy_async (a device-to-device cudaMemcpyAsync, done by
 * the copy engines) while the next chunk is updated.  `peers` (may be NULL)
 * are replicas the range's kernel stores to itself, as in the *_gather entry
 * points, so some peers can be served by the kernel and others by the copy
 * engines.
 */
int srs_adamw_multi_range(const srs_row* rows, int64_t n_rows, int64_t n_tiles, int64_t tile_lo,
                          int64_t tile_hi, int m_format, int m_rule, int v_format, int v_rule,
                          const srs_adamw_hparams* hp, const srs_rng* rng, uint32_t uniform_kind,
                          const srs_peers* peers, int grid_ctas, void* stream);

int srs_sgdm_multi_range(const srs_row* rows, int64_t n_rows, int64_t n_tiles, int64_t tile_lo,
                         int64_t tile_hi, int u_format, int u_rule, const srs_sgdm_hparams* hp,
                         const srs_rng* rng, uint32_t uniform_kind, const srs_peers* peers,
                         int grid_ctas, void* stream);

int srs_copy_async(void* dst, const void* src, uint64_t bytes, void* stream);

/* Peer mappings (CUDA IPC) of the buffers above.  srs_ipc_export writes a
 * handle of the allocation holding device address `p` (SRS_IPC_HANDLE_BYTES
 * bytes) and the offset of `p` inside it; srs_ipc_import maps a peer's
 * allocation into this process on the current device; srs_ipc_close unmaps
 * it.  Allocations from the virtual-memory API (expandable segments) cannot
 * be exported: srs_ipc_export then fails and the caller keeps a collective. */
#define SRS_IPC_HANDLE_BYTES 64
int srs_ipc_export(const void* p, void* handle, uint64_t* offset);
int srs_ipc_import(const void* handle, void** base);
int srs_ipc_close(void* base);

/* ---- multi-tensor AdamW step that allocates nothing ----------------------
 * No counterpart in the reference.  Same update as srs_adamw_multi, for
 * callers that cannot allocate device memory at step time (a runtime whose
 * allocator is reserved or already full, or a step issued from code that must
 * not call into any allocator).  `host_rows` is a HOST array of n_rows srs_row,
 * copied on `stream` into a fixed device-resident table of
 * SRS_NOALLOC_MAX_ROWS rows that every call on a device shares.  The copy is an
 * ordinary host-to-device cudaMemcpyAsync on `stream`: keep host_rows valid and
 * unchanged until the step has run on the stream.  The parameter/gradient
 * dtype kind is read from the rows.
 * Limits and rules:
 *   - n_rows > SRS_NOALLOC_MAX_ROWS fails with SRS_ERR_INVALID_ARGUMENT;
 *   - rows are checked on the host before anything is enqueued: tile_begin
 *     prefix sums, n_tiles, step classes, null addresses, and the alignment a
 *     row's SRS_ROW_VECTOR_OK flag promises (16 bytes for parameters,
 *     gradients and 2- or 4-byte states, 8 bytes for FP8 states); a violation
 *     fails with SRS_ERR_INVALID_ARGUMENT;
 *   - the first call on a device looks up the table's address (set-up); make
 *     that first call before any stream capture (a first call made during
 *     capture fails with SRS_ERR_INVALID_ARGUMENT);
 *   - a call captured into a CUDA graph captures the row copy too, which then
 *     reads host_rows at every replay: under capture host_rows must be
 *     page-locked (cudaHostAlloc / cudaHostRegister; pageable rows fail with
 *     SRS_ERR_INVALID_ARGUMENT) and stay valid while the graph can be
 *     replayed; a replay uses the rows' contents at that time, but the
 *     hyperparameters and RNG words captured with the call;
 *   - calls on one device that can overlap in time (different streams or host
 *     threads without ordering) race on the shared table: order them.
 */
#define SRS_NOALLOC_MAX_ROWS 4096
int srs_adamw_multi_noalloc(const srs_row* host_rows, int64_t n_rows, int64_t n_tiles,
                            int m_format, int m_rule, int v_format, int v_rule,
                            const srs_adamw_hparams* hp, const srs_rng* rng, int grid_ctas,
                            void* stream);

/* ---- fused single-tensor steps ------------------------------------------
 * Replace sr_states/triton/adamw.py:160-221 (`triton_adamw_step_`) and
 * sr_states/triton/sgd.py:115-171 (`triton_sgdm_step_`).  `row` is a HOST
 * srs_row describing one tensor; its param_index field holds the update key
 * (the functional API's `seed`).  hp->n_step_classes must be 1.
 */
int srs_adamw_single(const srs_row* row, int m_format, int m_rule, int v_format, int v_rule,
                     const srs_adamw_hparams* hp, int grid_ctas, void* stream);

int srs_sgdm_single(const srs_row* row, int u_format, int u_rule, const srs_sgdm_hparams* hp,
                    int grid_ctas, void* stream);

/* ---- RNG key derivation on the device ----------------------------------
 * Mirrors sr_states/triton/_keys.py:20-30 (_update_key/_state_key), used to
 * check that device keys equal host keys.  For each i < n writes
 * out[3i..3i+2] = {update_key(words, param_index[i]), state_key(k, 0), state_key(k, 1)}.
 */
int srs_derive_keys(const uint32_t* param_index, uint32_t* out, int64_t n, const srs_rng* rng,
                    void* stream);

/* ---- orthogonalised updates (Newton-Schulz) -------------------------------
 * No counterpart in the reference.  y = X_steps of
 *   X_0 = x / (|x|_F + eps);  X_{i+1} = (a I + b G + c G^2) X_i,  G = X_i X_i^T
 * for `batch` matrices of m rows and n columns (m > n: X_{i+1} = X_i (a I + b G + c G^2),
 * G = X_i^T X_i).  Products on the tensor cores with FP32 sums: FP16 operands for y in
 * BF16 (relative errors of the whole matrix of 1e-3 to 3e-3 whatever the singular values, of
 * 6e-3 for a few orthogonal rows and for ranks of a few at sides of ten thousand), pairs of
 * FP16 operands for y in FP32 or FP16 (1e-5 for sides of some hundreds, 1e-4 for ten thousand;
 * with ranks of a few 3e-4 and 3e-3; three times the work); the norm is summed in FP64.  Singular values must stay below 15
 * through the steps (those of the usual coefficients stay below 1.3).  x: FP32, BF16 or FP16, element (b, i, j) at
 * b * batch_stride + i * row_pitch + j; y: contiguous, FP32, BF16 or FP16; x and y must not
 * overlap.  At most 65535 matrices of 2^32 elements and 2^24 rows or columns.  A matrix with
 * a NaN or infinity, or whose norm plus eps is zero, gives NaN throughout.  Sizes of zero
 * are a no-op.
 * `workspace`: srs_newton_workspace(batch, m, n, y_format) bytes, 256-byte aligned, not used
 * by any other call that can overlap in time. */
#define SRS_NEWTON_MAX_STEPS 32
typedef struct srs_newton {
  int32_t steps;         /* 1..SRS_NEWTON_MAX_STEPS */
  float coefficients[3]; /* a, b, c */
  float eps;
} srs_newton;

int64_t srs_newton_workspace(int64_t batch, int64_t m, int64_t n, int y_format);

int srs_orthogonalize(const void* x, int x_format, int64_t row_pitch, int64_t batch_stride,
                      void* y, int y_format, int64_t batch, int64_t m, int64_t n,
                      const srs_newton* h, void* workspace, int64_t workspace_bytes,
                      void* stream);

/* Muon step of the matrices of up to SRS_MUON_MAX_CLASSES shapes (contiguous): per
 * element, each FP32 operation rounded once,
 *   u' = u*momentum + g;  v = nesterov ? u'*momentum + g : u'
 *   p' = fma(neg_step, O, p*decay),  O = the orthogonalised v of the matrix
 * u' is stored in u_format by u_rule (counter base state_key(key, 0), as the other
 * steps).  `rows`: HOST array, one row a matrix, read during the call: param, grad,
 * state[0], param_index, offset and flags are used and checked, numel and tile_begin are
 * not.  `classes`: HOST array; class i covers the next `count` rows, matrices of m x n,
 * count > 0, at most SRS_MUON_MAX_MATRICES rows in all.
 * neg_step = -(lr * the shape's factor), decay = 1 - lr*weight_decay.
 * `workspace`: srs_muon_workspace(classes, n_classes) bytes (-1: invalid classes). */
#define SRS_MUON_MAX_CLASSES 16
#define SRS_MUON_MAX_MATRICES 64
typedef struct srs_muon_class {
  int64_t count, m, n;
  float neg_step;
  int32_t reserved;
} srs_muon_class;

typedef struct srs_muon_hparams {
  float momentum, decay;
  int32_t nesterov;
} srs_muon_hparams;

int64_t srs_muon_workspace(const srs_muon_class* classes, int n_classes);

/* Side of the tiles in which a call with these matrices computes its products: 256 (two
 * CTAs a tile) or 128; negative: invalid sizes.  y_format as for srs_orthogonalize; Muon
 * steps take SRS_FMT_BF16. */
int srs_newton_tile(const srs_muon_class* classes, int n_classes, int y_format);

int srs_muon_multi(const srs_row* rows, const srs_muon_class* classes, int n_classes,
                   int u_format, int u_rule, const srs_muon_hparams* hp, const srs_newton* h,
                   const srs_rng* rng, void* workspace, int64_t workspace_bytes, void* stream);

/* ---- FP8 blocks and their products -----------------------------------------
 * No counterpart in the reference.  A matrix in FP8 blocks is `data` (E4M3 or
 * E5M2, rows x cols) with one power-of-two scale (UE8M0: byte b stands for
 * 2^(b-127)) for every 128 consecutive columns of a row (square == 0), or of every
 * 128 x 128 elements (square == 1); blocks at the edges hold what is left.
 *
 * srs_quantize_blocks: per block, k = the smallest exponent >= -127 with
 * max|finite x| <= largest * 2^k (0 for a block without nonzero finite values);
 * data = round(x * 2^-k) by `rule` (as srs_cast: infinities saturate, NaN is kept).
 * `data`/`scale`: of x; `data_t`/`scale_t`: of x transposed (cols x rows, blocks
 * along x's rows); either pair may be NULL.  Stochastic counters: element (i, j) of
 * x uses (i*cols + j + offset + state_key(seed, 0)) mod 2^32, its transposed copy
 * state_key(seed, 1).  x: FP32, BF16 or FP16, element (i, j) at i*x_pitch + j.  Row
 * pitches of data and data_t are in elements, those of scale and scale_t in blocks; the
 * copies' addresses and pitches are multiples of 16, and nothing is written outside their
 * rows and columns.  At most 4194240 rows and 2^30 columns a call.
 *
 * srs_matmul_blocks: d[i, j] = sum_k a[i, k] * b[j, k] with FP32 sums (terms truncated:
 * within (k + 2) 2^-23 of the sum of their sizes), k at most 2^30, d in FP32, BF16 or FP16
 * (contiguous).  The data's base addresses and row pitches must be
 * multiples of 16 bytes.  k == 0 gives zeros. */
int srs_quantize_blocks(const void* x, int x_format, int64_t rows, int64_t cols, int64_t x_pitch,
                        int out_format, int rule, int square, uint32_t seed, uint32_t offset,
                        void* data, int64_t data_pitch, void* scale, int64_t scale_pitch,
                        void* data_t, int64_t data_t_pitch, void* scale_t,
                        int64_t scale_t_pitch, void* stream);

/* Where a quantised copy goes: row pitches in elements and in blocks; in a stack, elements and
 * blocks from one matrix to the next. */
typedef struct srs_block_copy {
  uint64_t data, scale; /* device addresses; data == 0: no such copy */
  int64_t pitch, scale_pitch, stride, scale_stride;
} srs_block_copy;

/* A stack of at most 65535 matrices, each quantised as by srs_quantize_blocks; counters go on
 * from one matrix to the next: (b*rows + i)*cols + j. */
int srs_quantize_stack(const void* x, int x_format, int64_t matrices, int64_t rows, int64_t cols,
                       int64_t x_pitch, int64_t x_stride, int out_format, int rule, int square,
                       uint32_t seed, uint32_t offset, const srs_block_copy* copy,
                       const srs_block_copy* copy_t, void* stream);

typedef struct srs_blocks {
  uint64_t data;  /* device address, row pitch `pitch` bytes */
  uint64_t scale; /* device address, row pitch `scale_pitch` bytes */
  int64_t rows, pitch, scale_pitch;
  int32_t format; /* SRS_FMT_E4M3 or SRS_FMT_E5M2 */
  int32_t square; /* 1: one scale for 128 rows */
} srs_blocks;

int srs_matmul_blocks(const srs_blocks* a, const srs_blocks* b, int64_t k, void* d, int d_format,
                      void* stream);

/* d = x w^T: x (tokens x k, FP32, BF16 or FP16, row pitch x_pitch elements) quantised to
 * nearest in block_format (1 x 128 blocks) into `workspace` (srs_linear_workspace(tokens, k)
 * bytes, 16-byte aligned), times the blocks of w; d in x's format, contiguous tokens x
 * w->rows.  The same values as the two calls one after the other. */
int64_t srs_linear_workspace(int64_t tokens, int64_t k);
int srs_linear_blocks(const void* x, int x_format, int64_t tokens, int64_t k, int64_t x_pitch,
                      int block_format, const srs_blocks* w, void* d, void* workspace,
                      int64_t workspace_bytes, void* stream);

/* ---- rows in groups ---------------------------------------------------------
 * No counterpart in the reference.  Group g of `groups` (at most SRS_MAX_GROUPS) has rows
 * ends[g-1] .. ends[g] - 1 of a matrix (from 0 for the first); rows from the last end on
 * belong to none.  `ends` is in device memory; it is read as its running maximum, cut to
 * 0 .. rows, so that no value in it leads outside the matrix.
 *
 * srs_group_rows: stable sort of rows by their group.  index[i]: int32 (index_bytes 4) or int64
 * (8); values outside 0 .. groups - 1 mean no group.  order: the rows of group 0 in order, then
 * group 1's, .. , then those of none; ends[g]: rows with a group of at most g. */
#define SRS_MAX_GROUPS 1024
int srs_group_rows(const void* index, int index_bytes, int64_t rows, int groups, int32_t* order,
                   int32_t* ends, void* stream);

/* FP8 blocks of a matrix whose rows are in groups, for srs_expert_gradient: the transposed copy
 * in blocks of 128 rows counted from each group's first, srs_group_columns(rows, groups)
 * columns of data and srs_group_scales(rows, groups) scales a row (a layout of the library's
 * own, at a multiple of 4 bytes); beside it, on demand, the copy by rows.  Rows of no group are not written.  Counters are
 * those of srs_quantize_blocks. */
int64_t srs_group_columns(int64_t rows, int groups);
int64_t srs_group_scales(int64_t rows, int groups);
int srs_quantize_groups(const void* x, int x_format, int64_t rows, int64_t cols, int64_t x_pitch,
                        const int32_t* ends, int groups, int out_format, int rule, uint32_t seed,
                        uint32_t offset, const srs_block_copy* copy, const srs_block_copy* copy_t,
                        void* stream);

/* d[i, :] = a[i, :] w_e^T for the rows i of group e; zeros for rows of none.  a: rows x k;
 * w: `experts` matrices of n x k one after the other (w->rows = experts * n; square blocks start
 * anew with every matrix); d: a->rows x n, contiguous.  Sums and limits as srs_matmul_blocks.
 * experts * n is at most 2^30. */
int srs_expert_matmul(const srs_blocks* a, const srs_blocks* w, int experts, const int32_t* ends,
                      int64_t k, void* d, int d_format, void* stream);

/* The same of x quantised to nearest in block_format (1 x 128 blocks) into `workspace`
 * (srs_linear_workspace(rows, k) bytes, 16-byte aligned); d in x's format. */
int srs_expert_linear(const void* x, int x_format, int64_t rows, int64_t k, int64_t x_pitch,
                      int block_format, const srs_blocks* w, int experts, const int32_t* ends,
                      void* d, void* workspace, int64_t workspace_bytes, void* stream);

/* d_e = a_e^T b_e for every group e: a_t and b_t are the transposed copies (srs_quantize_groups)
 * of two matrices of `rows` rows, m x rows and n x rows; d: experts x m x n, contiguous; zeros
 * for groups without rows. */
int srs_expert_gradient(const srs_blocks* a_t, const srs_blocks* b_t, int64_t rows, int experts,
                        const int32_t* ends, void* d, int d_format, void* stream);

/* ---- low-rank adapters beside a projection in FP8 blocks -----------------------
 * No counterpart in the reference.  Token t has adapter a, the group that order and ends
 * (srs_group_rows) give it, or none.  16-bit matrices `down` (count x rank x in) and `up`
 * (count x out x rank); addresses, row pitches and strides are multiples of 16 bytes; a row's
 * elements follow one another.  scale: FP32, one an adapter (0: none), times `factor`.
 *
 * srs_adapter_linear: with x (tokens x k, in the adapters' format) quantised in 1 x 128 blocks of
 * block_format by `rule` and `seed`,
 *   turned == 0:  low_t = s_a down_a x_t;    d_t = w x_t + up_a low_t        (k = in, w->rows = out)
 *   turned == 1:  low_t = s_a up_a^T x_t;    d_t = w x_t + down_a^T low_t    (k = out, w->rows = in)
 * Sums of both parts in FP32, d (tokens x w->rows, in the adapters' format) rounded once.  low:
 * FP32, tokens (in the order of `order`) x rank, or NULL; rows of tokens without an adapter are
 * not written.  largest (FP16 alone): `count` words, encodings of max |low| of every adapter, or
 * NULL.  d == NULL: `low` alone.
 *
 * srs_adapter_gradient: one or two sums over the tokens of every adapter, out_a = sum of low_t
 * z_t^T (rank x cols) or, turned, z_t low_t^T (cols x rank), in z's format; zeros without tokens.
 * `largest` as given above (FP16).  The workspace is that of all sums' columns together.
 *
 * `workspace`: 256-byte aligned, not used by any other call that can overlap in time. */
#define SRS_ADAPTER_MAX_RANK 256
typedef struct srs_adapters {
  uint64_t down, up, scale, order, ends; /* device addresses */
  int64_t down_pitch, down_stride, up_pitch, up_stride; /* elements */
  float factor;
  int32_t count, rank, format;
} srs_adapters;

int64_t srs_adapter_workspace(int64_t tokens, int64_t k, int64_t n, int adapters, int rank);
int srs_adapter_linear(const void* x, int64_t tokens, int64_t k, int64_t x_pitch,
                       int block_format, int rule, uint32_t seed, const srs_blocks* w,
                       const srs_adapters* a, int turned, void* d, float* low, uint32_t* largest,
                       void* workspace, int64_t workspace_bytes, void* stream);

int64_t srs_adapter_gradient_workspace(int64_t tokens, int64_t cols, int adapters, int rank);
typedef struct srs_adapter_sum {
  uint64_t z; /* tokens x cols, 16-byte aligned, row pitch z_pitch elements */
  int64_t z_pitch, cols;
  uint64_t low, largest, out; /* low: 16-byte aligned */
  int64_t turned;
} srs_adapter_sum;
int srs_adapter_gradient(const srs_adapter_sum* sums, int n_sums, int format, int64_t tokens,
                         int adapters, int rank, const int32_t* order, const int32_t* ends,
                         void* workspace, int64_t workspace_bytes, void* stream);

/* Rows of `cols` bytes at src_pitch copied to rows at dst_pitch (zeros behind them up to
 * dst_pitch): for operands whose rows do not start on 16-byte boundaries.  dst and
 * dst_pitch must be multiples of 16 bytes. */
int srs_copy_rows(const void* src, int64_t src_pitch, int64_t rows, int64_t cols, void* dst,
                  int64_t dst_pitch, void* stream);

/* Waits inside the product kernels are bounded (about 2 s beyond what their work takes).  One that runs out is recorded
 * in a word of host memory, one a device, and the results of that call are not valid (a
 * Muon step's parameters and momentum neither).  The next srs_orthogonalize,
 * srs_muon_multi, srs_matmul_blocks or srs_linear_blocks on the device enqueues nothing,
 * clears the word and returns SRS_ERR_WAIT.
 * srs_product_status: synchronises the current device, gives the word (0: no wait ran out
 * since it was last cleared) and clears it.
 * srs_product_status_word: the word's host address, to look at without synchronising. */
int srs_product_status(uint32_t* status);
int srs_product_status_word(uint32_t** word);

#ifdef __cplusplus
}
#endif

#endif /* SRS_B200_H */
