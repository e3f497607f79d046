/*
 * vmonarch_b200 — C ABI of the B200 (sm_100a) VMonarch attention hot path.
 *
 * The reference (EricLina/VMonarch) is a Python package whose hot path crosses from the host to
 * the GPU only at its Triton kernel launches and at a handful of torch ops. Each entry point
 * below replaces one of those crossings; the Python package `vmonarch_b200` binds them with
 * ctypes and mirrors the reference's Python API on top.
 *
 * Conventions
 *  - Every pointer is a device pointer; tensors are dense row-major with the batch stride given
 *    in ELEMENTS. Rows are contiguous (row stride = number of columns). Base pointers must be
 *    16-byte aligned and batch strides multiples of 8 elements.
 *  - dtype selects the 16-bit element type (VMB_DTYPE_BF16 or VMB_DTYPE_F16); all arithmetic
 *    accumulates in fp32. Statistics (lse, ent, dent) are fp32.
 *  - `stream` is a cudaStream_t (NULL = legacy default stream). Calls only enqueue work; they
 *    never synchronize and never allocate.
 *  - Return value: VMB_OK or an error code; vmb_last_error() describes the last failure of the
 *    calling thread.
 */
#ifndef VMONARCH_B200_H
#define VMONARCH_B200_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define VMB_ABI_VERSION 7

#define VMB_DTYPE_BF16 0
#define VMB_DTYPE_F16 1

#define VMB_OK 0
#define VMB_EINVAL 1   /* malformed argument: null pointer, bad size, misalignment */
#define VMB_ENOTSUP 2  /* head dimensions without a kernel, or a strided layout a kernel cannot take */
#define VMB_ECUDA 3    /* CUDA runtime error while launching */

/* ABI version (VMB_ABI_VERSION of the library that was loaded). */
int vmb_abi_version(void);

/* Human-readable description of the last error returned on the calling thread. */
const char* vmb_last_error(void);

/* Pipeline-timeout status of the tcgen05 kernels on the current device: synchronises `stream`,
 * stores into *out the OR of the error codes recorded since the last call (0 = none) and clears
 * them. A kernel whose pipeline wait exceeds its time limit (~2 s) records a code, drains its
 * in-flight copies and MMAs, frees its tensor memory and exits instead of hanging; its outputs
 * are then invalid. No counterpart in the reference (Triton kernels have no such check). */
int vmb_device_status(void* stream, int32_t* out);

/* Test hook of the pipeline-timeout path; no counterpart in the reference. wait_cycles > 0
 * shortens the pipeline wait limit of the tcgen05 forward kernels and of the packed and paged attention
 * kernels to that many SM cycles; hold_loads != 0 (only with 0 < wait_cycles <= 1e8) makes their
 * load producers (paged: one of a block's four warps) issue no copy, so the consumers' first waits
 * run out: the kernels record their codes (vmb_device_status), drain, free their tensor memory and
 * exit with their outputs invalid. (0, 0) restores normal operation. The setting is process-wide and
 * read at each vmb_fea_fwd, vmb_packed_fwd, vmb_packed_bwd and vmb_paged_attention call; it exists
 * for tests only. */
int vmb_test_pipeline_timeout(int64_t wait_cycles, int32_t hold_loads);

/* Number of kernels this library has launched in the process so far (all threads, all devices).
 * Diagnostic with no reference counterpart: the benchmark reports it as its launch count. */
uint64_t vmb_kernel_launches(void);

/*
 * Strided layouts (ABI version 6). By default every tensor is dense [batch][rows][cols] with the
 * batch stride given in its *_bs field. A call may instead pass a layout that gives each tensor a
 * view: element (s, r, c) of batch entry s, row r, column c lies at
 *     c + r * row + (s % n1) * s1 + (s / n1 % n2) * s2 + (s / (n1 * n2)) * s3
 * elements from the tensor's base, with (n1, n2) shared by the call's tensors (batch must be a
 * multiple of n1 * n2). This is how token-major callers are served without transposes: the
 * reference's Video-DiT caller holds tokens as (B, N, H, D) (README.md:74-76), whose head h of
 * batch b is rows of stride H * D starting at (b * N * H + h) * D, so FlashEntropyAttention over
 * its B * H sequences is the view {H * D, D, 0, N * H * D} with (n1, n2) = (H, 1), and the VMonarch
 * R step over its B * H * m grid rows of b tokens is {H * D, b * H * D, D, N * H * D} with
 * (n1, n2) = (m, H). Strides are in elements and multiples of 8 (4 for fp32 tensors); row >= cols.
 * Statistics (lse, ent, dent, delta) stay dense [batch][rows] in every layout. Only the D = 128
 * kernels take non-uniform views (a view is uniform when row == cols and entry s starts at s * X);
 * other head dimensions return VMB_ENOTSUP for them.
 */
typedef struct vmb_view {
  int64_t row, s1, s2, s3;
} vmb_view;

typedef struct vmb_fea_layout {
  int64_t n1, n2;
  vmb_view q, k, v, v2, o, dout, grad_q, grad_k, grad_v, grad_v2, fin_q, fin_k, fin_v, fin_v2;
} vmb_fea_layout;

/*
 * FlashEntropyAttention forward over `batch` independent sequences:
 *   o = softmax(sm_scale q k^T) [v | v2],  ent_i = -sum_j P_ij log P_ij,
 *   lse_i = log2 sum_j 2^(x_ij) with x = sm_scale q k^T log2(e)   (kept for the backward).
 * Replaces the `_attn_fwd` launch and the pad-row zeroing of _FlashEntropyAttention.forward
 * (video_monarch_attention/kernel.py:346-353) and the F.pad / slice of flash_entropy_attention
 * (kernel.py:399-402): sequences of any length are handled without padding. The optional second
 * value tensor replaces the torch.cat([kg, vg], -1) of the last R step (vmonarch.py:50).
 * Shapes: d, dv in {16, 32, 64, 128, 256} with dv a multiple of d (the reference requires
 * Dv % D == 0 for its backward, kernel.py:260). o may be a strided view (o_bs) into a larger
 * tensor, which is how the exact first-frame recompute writes straight into z.
 * workspace / workspace_bytes are optional (NULL / 0 is valid). With a workspace of
 * vmb_fea_fwd_workspace_bytes() bytes the d = dv = 128 kernel may split each sequence's key range
 * over several CTAs when the query tiles alone would fill the GPU poorly (few, long sequences, e.g.
 * the recompute's r queries over all N keys on a few heads); the partial results are merged
 * exactly by a second kernel. Without one, or when no split pays off, nothing changes. The
 * workspace contents need not be initialised; it is 256-byte aligned when obtained from a
 * caching allocator (16 bytes is required).
 */
typedef struct vmb_fea_fwd_args {
  const void* q;  int64_t q_bs;   /* [batch][n_q][d]                               */
  const void* k;  int64_t k_bs;   /* [batch][n_kv][d]                              */
  const void* v;  int64_t v_bs;   /* [batch][n_kv][dv1]  -> o columns [0, dv1)     */
  const void* v2; int64_t v2_bs;  /* [batch][n_kv][dv-dv1] -> o columns [dv1, dv); NULL if dv1 == dv */
  void* o;        int64_t o_bs;   /* [batch][n_q][dv]                              */
  float* lse;                     /* [batch][n_q] or NULL                          */
  float* ent;                     /* [batch][n_q] or NULL (entropy not computed)   */
  int64_t batch, n_q, n_kv;
  int32_t d, dv, dv1, dtype;
  float sm_scale;
  void* workspace;  int64_t workspace_bytes;  /* optional, see above (ABI version 2) */
  const vmb_fea_layout* layout;  /* optional strided layout of q, k, v, v2, o (ABI version 6);
                                    NULL: dense with the *_bs batch strides */
  int32_t qkv_e4m3;  /* ABI version 7. Nonzero: q, k, v and v2 hold e4m3 (fp8, one byte per
                        element; see vmb_quant_e4m3) and both products run on the fp8 tensor cores,
                        with P rounded to e4m3 as well; o, lse and ent are as usual (dtype gives o's
                        type). Only the VMonarch R-step forms: d = 128, v aliasing k (v == k, dv1 = d),
                        dv = 128 or dv = 256 with a 128-wide v2. Batch and layout strides are then
                        multiples of 16 elements (bytes). No reference counterpart: an opt-in
                        B200 extension of the R step (the reference computes it in bf16). */
} vmb_fea_fwd_args;

/* Workspace that lets vmb_fea_fwd split long key ranges (0 when it would not split). No
 * counterpart in the reference, whose forward launch allocates through torch. */
int64_t vmb_fea_fwd_workspace_bytes(const vmb_fea_fwd_args* a);
int vmb_fea_fwd(const vmb_fea_fwd_args* a, void* stream);

/*
 * FlashEntropyAttention backward. Replaces `_attn_bwd_preprocess` + `_attn_bwd`
 * (video_monarch_attention/kernel.py:360-381) including the entropy-gradient term
 * dS = P (dP - delta) + dE P (-E - log P) (kernel.py:165-167).
 * grad_mode 0: grad_q/grad_k/grad_v/grad_v2 are written in the element dtype (standalone op).
 * grad_mode 1: grad_* are fp32 buffers that the gradients are ADDED into (VMonarch chains
 *              several R steps and the recompute into one set of accumulators).
 * grad_mode 2: grad_* are fp32 buffers that are OVERWRITTEN (the first contribution to a set of
 *              accumulators, so they need no zero-fill).
 * grad_mode 3: the last contribution: grad_* are written in the element dtype as the sum of the
 *              fp32 accumulator fin_* (same shape, batch stride fin_*_bs) and this call's gradient,
 *              which saves a separate fp32 -> 16-bit pass. fin_q/fin_k (and fin_v / fin_v2 where
 *              grad_v / grad_v2 are given) are required; their contents are unspecified afterwards
 *              (shapes without a tcgen05 kernel add into them before converting).
 * v_is_k = 1: the value columns [0, dv1) are the key tensor itself (dv1 == d); their gradient is
 *              added into grad_k and grad_v must be NULL. This is the VMonarch R step
 *              (vmonarch.py:50).
 * dent may be NULL (dE = 0, e.g. the detached entropy of VMonarch, vmonarch.py:26); ent is then
 * not read either.
 * The caller provides a device workspace of vmb_fea_bwd_workspace_bytes() bytes (256-byte
 * aligned); its contents need not be initialised.
 */
typedef struct vmb_fea_bwd_args {
  const void* q;    int64_t q_bs;
  const void* k;    int64_t k_bs;
  const void* v;    int64_t v_bs;
  const void* v2;   int64_t v2_bs;
  const void* o;    int64_t o_bs;    /* forward output                         */
  const void* dout; int64_t do_bs;   /* gradient of o, [batch][n_q][dv]        */
  const float* lse;                  /* forward lse, [batch][n_q]              */
  const float* ent;                  /* forward entropy (read only with dent)  */
  const float* dent;                 /* gradient of ent or NULL                */
  void* grad_q;  int64_t grad_q_bs;   /* [batch][n_q][d]                        */
  void* grad_k;  int64_t grad_k_bs;   /* [batch][n_kv][d]                       */
  void* grad_v;  int64_t grad_v_bs;   /* [batch][n_kv][dv1]  (NULL if v_is_k)   */
  void* grad_v2; int64_t grad_v2_bs;  /* [batch][n_kv][dv-dv1] (NULL if no v2)  */
  void* workspace; int64_t workspace_bytes;
  int64_t batch, n_q, n_kv;
  int32_t d, dv, dv1, dtype;
  int32_t grad_mode, v_is_k;
  float sm_scale;
  const float* delta;  /* optional [batch][n_q] fp32: sum_c o[c] dout[c] per query row, precomputed
                          by the caller (vmb_lstep_bwd's delta_out); NULL: computed here (ABI 2) */
  int32_t deterministic; /* nonzero: bitwise reproducible gradients. Zero lets grad_mode 1 / 2 with
                            v_is_k, dv == d == 128 and n_kv <= 4096 form dQ with concurrent fp32
                            reductions (one kernel fewer; summation order varies) (ABI 3) */
  const float* fin_q;  int64_t fin_q_bs;   /* grad_mode 3 accumulators (ABI 4) */
  const float* fin_k;  int64_t fin_k_bs;
  const float* fin_v;  int64_t fin_v_bs;
  const float* fin_v2; int64_t fin_v2_bs;
  const vmb_fea_layout* layout;  /* optional strided layout of every tensor but the statistics
                                    (ABI version 6); NULL: dense with the *_bs batch strides */
} vmb_fea_bwd_args;

int64_t vmb_fea_bwd_workspace_bytes(const vmb_fea_bwd_args* a);
/* The smallest workspace vmb_fea_bwd accepts (ABI 5). vmb_fea_bwd_workspace_bytes reports the
 * preferred size, which for the last VMonarch R step (v_is_k, dv = 2 d, n_kv <= 4096) adds a dS^T
 * buffer (batch x round_up(n_kv, 128) x round_up(n_q, 64) 16-bit values) so that dQ comes from
 * dS by a GEMM instead of a kernel recomputing S and dP; a workspace between the two sizes runs
 * the latter. -1 for malformed sizes. */
int64_t vmb_fea_bwd_min_workspace_bytes(const vmb_fea_bwd_args* a);
int vmb_fea_bwd(const vmb_fea_bwd_args* a, void* stream);

/*
 * vmb_fea_bwd for callers that cannot allocate device memory. No counterpart in the reference.
 * Same arguments and results as vmb_fea_bwd, but `workspace` / `workspace_bytes` are ignored: the
 * scratch comes from a 32 MiB array compiled into the library (a static __device__ buffer that
 * every GPU holding the library's module keeps until the process exits). Meant for hosts that
 * cannot hand over a workspace: plugins whose enqueue hook must not allocate because the host
 * framework owns all device memory, foreign-language bindings that can only pass the user's
 * tensors, and pipelines that cannot afford cudaMalloc inside a step.
 *  - Calls whose minimal workspace (vmb_fea_bwd_min_workspace_bytes) exceeds 32 MiB return
 *    VMB_EINVAL. A call whose preferred workspace (vmb_fea_bwd_workspace_bytes, which adds the
 *    dS^T buffer of the dQ-from-dS route) also fits takes that route; otherwise it runs the dQ
 *    kernel that recomputes S and dP, with the same results.
 *  - The first call on a device looks the buffer's address up with that device current; make
 *    that first call before any stream capture begins. The address is kept for the process: after
 *    cudaDeviceReset (which unloads the library's module) or from a context other than the
 *    device's primary context this entry point must not be used.
 *  - All calls share the buffer, which keeps the previous call's contents (the backward clears
 *    what must start at zero). Calls that overlap on the GPU race on it: serialise them.
 *  - Calls no cudaMalloc, cudaFree or other allocating routine.
 */
int vmb_fea_bwd_noalloc(const vmb_fea_bwd_args* a, void* stream);

/*
 * Monarch L step (the b dense m x m blocks), forward and backward, for `bh` heads of
 * N = m * b tokens. Replaces the einsum / softmax / col_mass / scaling ops of
 * video_monarch_attention/vmonarch.py:51-63 (forward) and their autograd backward.
 *   q    [bh][N][d]   original queries        out [bh][N][dw] R-step output
 *   ent  [bh][N]      R-step row entropy (the reference's -neg_ent)
 * forward, last == 0: u  [bh][N][d]    next R-step queries (already scaled)
 * forward, last == 1: z  [bh][N][dw-d] Monarch output; tokens < skip_rows are left unwritten
 * backward, last == 0: du [bh][N][d] fp32 gradient of u
 * backward, last == 1: dz [bh][N][dw-d] gradient of z; tokens < skip_rows carry none
 * backward outputs: dq [bh][N][d] fp32 (ADDED into, or OVERWRITTEN when dq_store != 0),
 *   dout [bh][N][dw] gradient of out.
 * m <= 128 (m <= 64 unless d in {64, 128} with dw = d, or 2d when last), d in {16, 32, 64, 128},
 * dw - d in {16, ..., 256} and a multiple of d when last.
 */
/* Strided layout of an L-step call (ABI version 6): each tensor is a [bh][N][cols] view (rows =
 * tokens) whose head hb starts at (hb % n1) * s1 + (hb / n1) * s3 (s2 unused); a token-major
 * (B, N, H, D) tensor is {H * D, D, 0, N * H * D} with n1 = H. ent and delta_out stay dense. The
 * kernels for m <= 128 with d in {64, 128} take any view; other shapes need dense tensors. */
typedef struct vmb_lstep_layout {
  int64_t n1;
  vmb_view q, out, u, z, du, dz, dq, dout;
} vmb_lstep_layout;

typedef struct vmb_lstep_args {
  const void* q;
  const void* out;
  const float* ent;
  void* u;
  void* z;
  const float* du;
  const void* dz;
  float* dq;
  void* dout;
  int64_t bh, m, b;
  int32_t d, dw, dtype, last;
  int64_t skip_rows;
  float scale, min_col_mass;
  int32_t dq_store;  /* backward: 1 = write dq instead of adding into it (ABI version 2) */
  float* delta_out;  /* backward, optional [bh][N] fp32: sum_c out[c] dout[c] per token, the
                        preprocessing of the R step's attention backward (its `delta`) */
  const vmb_lstep_layout* layout;  /* optional (ABI version 6), see above; NULL: dense */
} vmb_lstep_args;


int vmb_lstep_fwd(const vmb_lstep_args* a, void* stream);
int vmb_lstep_bwd(const vmb_lstep_args* a, void* stream);

/* dst[b][i] = (dtype) src[b][i], i < n (n and both batch strides multiples of 4).
 * Converts the fp32 gradient accumulators of grad_mode 1 to the element dtype. */
int vmb_cast_f32(const float* src, int64_t src_bs, void* dst, int64_t dst_bs, int64_t batch, int64_t n,
                 int32_t dtype, void* stream);

/* dst(s, r, c) = e4m3(scale * src(s, r, c)) over [batch][rows][cols] views with batch split (n1, n2)
 * (ABI version 7): the operands of an e4m3 forward (vmb_fea_fwd_args.qkv_e4m3) from 16-bit tensors
 * of element type dtype. Rounded to nearest even, saturating at +-448 (the format's largest finite
 * value); NaN stays NaN. cols a multiple of 16; src rows 16-byte aligned (view strides multiples of
 * 8 elements), dst rows 16-byte aligned (multiples of 16). */
int vmb_quant_e4m3(const void* src, const vmb_view* src_view, void* dst, const vmb_view* dst_view, int64_t n1,
                   int64_t n2, int64_t batch, int64_t rows, int64_t cols, int32_t dtype, float scale, void* stream);

/* dst(s, r, c) = (dtype) src(s, r, c) over [batch][rows][cols] views with batch split (n1, n2)
 * (ABI version 6): the fp32 accumulator of a strided (e.g. token-major) gradient converted into
 * the caller's tensor. cols a multiple of 4; src rows 16-byte aligned, dst rows 8-byte aligned. */
int vmb_cast_f32_view(const float* src, const vmb_view* src_view, void* dst, const vmb_view* dst_view, int64_t n1,
                      int64_t n2, int64_t batch, int64_t rows, int64_t cols, int32_t dtype, void* stream);

/*
 * Attention over packed sequences of different lengths (no reference counterpart): the rows of q
 * (q_total x heads x dim) and of k, v (k_total x kv_heads x dim) hold the sequences one after
 * another; query head h reads key / value head h / (heads / kv_heads). With `causal`, local query i of
 * a sequence of nq queries and nk keys sees its first nk - nq + i + 1 keys. A query that sees no
 * key has o = 0, lse = -inf and passes no gradient. dim: a multiple of 8, at most 128.
 *
 * The work is described by units built on the host from the sequence lengths, in device memory
 * (int32, 48 bytes each). They are trusted: q_row + q_valid <= q_total, k_row + k_valid <= k_total.
 *  units    (forward) at most 256 queries of one sequence, key tiles [begin, end) of 128 keys
 *  q_units  (backward, dQ) the same with at most 128 queries
 *  kv_units (backward, dK / dV) at most 128 keys; k_row / k_valid are theirs, q_row / q_valid the whole
 *           sequence's queries, vis0 the local query that first sees the unit's key 0 (a large
 *           negative number when not causal); [begin, end) steps over (head of the group, 64-query
 *           tile from max(vis0, 0) / 64 on), heads outermost
 * For the first two, vis0 is the number of keys that local query 0 of the unit sees, before the limits
 * 0 and k_valid, and k_row / k_valid are the sequence's keys. stat_row: first row of the unit's
 * queries (kv_units: of the sequence's) in the backward's statistics, where every sequence starts
 * at a multiple of 128; stat_rows is their total. part: -1, or the slot (0 .. n_parts - 1) of a
 * piece of work that is split over its key tiles (dQ, forward) or steps (dK / dV); the pieces of a
 * split unit take consecutive slots, and `joins` lists them as (first unit, number of pieces). lone
 * (kv_units): the sequence's queries below it see one key at most, so their dS is zero; 0 where that is
 * not known. extra: 0. pieces: the host's own.
 */
typedef struct vmb_packed_unit {
  int32_t q_row, q_valid, k_row, k_valid, vis0, begin, end, part, stat_row, pieces, lone, extra;
} vmb_packed_unit;

typedef struct vmb_packed_list {
  const vmb_packed_unit* units;  /* device */
  const int32_t* joins;          /* device, (first unit, pieces) pairs; NULL when nothing is split */
  int32_t n_units, n_joins, n_parts, reserved;
} vmb_packed_list;

typedef struct vmb_rows {  /* [rows][heads][dim] view: strides of a row and of a head, in elements */
  void* ptr;
  int64_t row, head;
} vmb_rows;

typedef struct vmb_packed_args {
  vmb_rows q, k, v, o;       /* o: written by the forward, read by the backward     */
  vmb_rows dout, dq, dk, dv; /* backward                                            */
  vmb_rows o_low;            /* what o's rounding left out: 16-bit (exact o - o), written by the forward
                                where ptr is not NULL, required by the backward, whose sums o . dout
                                need more of o than its own 16 bits */
  float* lse;                /* [heads][q_total] natural log; NULL allowed (forward) */
  int64_t q_total, k_total, stat_rows;
  int32_t heads, kv_heads, dim, dtype, causal;
  float sm_scale;            /* >= 0 */
  vmb_packed_list units, q_units, kv_units;
  void* workspace; int64_t workspace_bytes;  /* 256-byte aligned */
} vmb_packed_args;

/* Workspace of vmb_packed_fwd (0 unless units are split) and of vmb_packed_bwd; -1: malformed. */
int64_t vmb_packed_fwd_workspace_bytes(const vmb_packed_args* a);
int64_t vmb_packed_bwd_workspace_bytes(const vmb_packed_args* a);
int vmb_packed_fwd(const vmb_packed_args* a, void* stream);
int vmb_packed_bwd(const vmb_packed_args* a, void* stream);
/* The same with a window (causal only): of the keys below its limit n a query sees the last `window` >= 1 and the first
 * `sinks` >= 0. units and q_units leave out the key tiles between the first sinks and the window of the unit's first
 * query: tile x of [begin, end) is key tile x below lone (the tiles of the sinks; 0 where nothing is left out) and
 * x + extra from there on. kv_units: the unit's first `extra` keys are sinks; without any the steps of a head end at the
 * tile of the last query that sees the unit's last key (local query vis0 + k_valid - 2 + window). lone there: all of
 * the sequence's queries where window + sinks is 1. */
int vmb_packed_window_fwd(const vmb_packed_args* a, int32_t window, int32_t sinks, void* stream);
int vmb_packed_window_bwd(const vmb_packed_args* a, int32_t window, int32_t sinks, void* stream);

/*
 * Paged key / value caches (no reference counterpart). A pool holds num_pages >= 1 pages of page_size slots;
 * a page of one tensor is [kv_heads][page_size][dim], anywhere its strides put it (elements, multiples
 * of 8; 16-byte aligned base). dim: a multiple of 8, at most 128.
 */
typedef struct vmb_pages {
  void* ptr;
  int64_t page, head, slot;  /* strides in elements */
} vmb_pages;

/* Attention of one new token per sequence: q, o [batch][heads][dim]; token t of sequence b lies in slot
 * t % page_size of page table[b * table_stride + t / page_size], t < lengths[b]. A sequence of length 0
 * has o = 0, lse = -inf. Lengths above table_width * page_size are cut to it and page ids outside the
 * pool read as zeros (their content is on the device, where a call cannot refuse it). */
typedef struct vmb_paged_args {
  vmb_rows q, o;
  vmb_pages k, v;
  const int32_t* table;    /* [batch][table_stride], device */
  const int32_t* lengths;  /* [batch], device */
  float* lse;              /* [batch][heads] natural logarithm, or NULL */
  int64_t batch, table_stride, table_width, num_pages;
  int32_t heads, kv_heads, dim, page_size, dtype;
  float sm_scale;
  void* workspace; int64_t workspace_bytes;  /* 256-byte aligned, of vmb_paged_workspace_bytes */
} vmb_paged_args;

int64_t vmb_paged_workspace_bytes(const vmb_paged_args* a);  /* -1: malformed sizes */
int vmb_paged_attention(const vmb_paged_args* a, void* stream);

/* One value per page and key head, device: value x scale[page * s.page + head * s.head]. */
typedef struct vmb_page_scales {
  float* ptr;
  int64_t page, head;
} vmb_page_scales;

/* The same over other caches: with a window a sequence's new token sees the last `window` >= 1 of its tokens and the first
 * `sinks` >= 0 (window 0: all, sinks 0), and table entries of pages without a token that it sees are not read. With
 * k_scale.ptr and v_scale.ptr the pools hold e4m3 values (one byte an element; dim and strides multiples of 16) with a scale
 * for each page and head, not negative; q and o stay of type dtype. NULL, both of them: 16-bit pools. */
typedef struct vmb_cache_args {
  vmb_page_scales k_scale, v_scale;
  int32_t window, sinks;
} vmb_cache_args;
int64_t vmb_cache_workspace_bytes(const vmb_paged_args* a, const vmb_cache_args* c);  /* -1: malformed sizes */
int vmb_cache_attention(const vmb_paged_args* a, const vmb_cache_args* c, void* stream);

/* Row i of k_new, v_new [count][kv_heads][dim] into slot slots[i] % page_size of page
 * slots[i] / page_size of each pool. Slots outside the pool (negative ones: padding) are skipped; no slot may be
 * named twice. 16-bit elements of any kind. */
int vmb_append_pages(const vmb_rows* k_new, const vmb_rows* v_new, const vmb_pages* k, const vmb_pages* v,
                     const int32_t* slots, int64_t count, int64_t num_pages, int32_t kv_heads, int32_t dim,
                     int32_t page_size, void* stream);
/* Page src[i] to page dst[i], i < count, in both pools. Pairs with a page outside the pool are skipped; no
 * destination may be another pair's source or destination. */
int vmb_copy_pages(const vmb_pages* k, const vmb_pages* v, const int32_t* src, const int32_t* dst, int64_t count,
                   int64_t num_pages, int32_t kv_heads, int32_t dim, int32_t page_size, void* stream);
/* The same for pools of e4m3 values with scales (vmb_cache_args). Appended rows are of type dtype. For every page, head and
 * tensor, the call's rows need the least power of two s, 2^-126 at least, with |x| <= 448 s for each of their finite values.
 * A call that writes slot 0 of a page begins it: its scale becomes s, and what its other slots held is void. Otherwise the
 * scale becomes the larger of s and what it was, and where it grows the page's other slots are brought to it (rounded to
 * nearest). Rows are divided by the scale and rounded to nearest even; infinities and NaN become NaN. The rows that go into
 * one page have to follow one another in the call, skipped ones not between them. */
typedef struct vmb_move_e4m3_args {
  vmb_rows k_new, v_new;             /* append */
  vmb_pages k, v;
  vmb_page_scales k_scale, v_scale;
  const int32_t *src, *dst;          /* copy: pages; append: dst are the slots */
  int64_t count, num_pages;
  int32_t kv_heads, dim, page_size, dtype;  /* dtype: of appended rows */
} vmb_move_e4m3_args;
int vmb_append_pages_e4m3(const vmb_move_e4m3_args* a, void* stream);
int vmb_copy_pages_e4m3(const vmb_move_e4m3_args* a, void* stream);

/*
 * The book of a paged cache on the device (no reference counterpart): sequence b of lengths[b] tokens holds
 * ceil(lengths[b] / page_size) pages, the first entries of its table row; free_pages[0 .. *num_free) is the stack of the
 * others. reserve: counts[b] more tokens of every sequence. The new pages of the sequences, in order, are taken from the
 * stack's end, lengths and *num_free follow, and slots[total] gets the slot of every new token, sequence after sequence, then
 * -1. truncate: every sequence keeps its first keep[b] tokens (negative: none); the pages beyond go back in the opposite order.
 * A call that cannot be done changes nothing, adds bits to *failed (1 too few free pages, 2 a table row too narrow, 4 more
 * tokens than rows or a negative number, 8 more pages than the stack has room for) and gives slots of -1.
 */
typedef struct vmb_page_book {
  int32_t* table;       /* [batch][table_stride], of which table_width entries a row */
  int32_t* lengths;     /* [batch] */
  int32_t* free_pages;  /* [num_pages] */
  int32_t* num_free;    /* [1] */
  int32_t* failed;      /* [1], or NULL */
  int64_t table_stride, batch, table_width, num_pages;
  int32_t page_size;
} vmb_page_book;

/* Workspace of either call; needed above 1024 sequences, for reserve above 4096 rows, for truncate above 65536 table entries. */
int64_t vmb_page_book_workspace_bytes(const vmb_page_book* b);  /* -1: malformed sizes */
int vmb_reserve_pages(const vmb_page_book* b, const int32_t* counts, int32_t* slots, int64_t total, void* workspace,
                      int64_t workspace_bytes, void* stream);
int vmb_truncate_pages(const vmb_page_book* b, const int32_t* keep, void* workspace, int64_t workspace_bytes, void* stream);

/*
 * Gated residual with norms around a block (no reference counterpart), over rows of `cols` elements that
 * belong to `seqs` sequences one after another (seq_start[s]: first row of sequence s, device int32;
 * NULL with one sequence):
 *   y^ = y / sqrt(mean(y^2) + eps) * post_weight   (without post_weight: y)
 *   x_new = x + gate y^,   h = norm(x_new) weight (1 + scale) + shift
 * norm: x / sqrt(mean(x^2) + eps), or with `layer` (x - mean) / sqrt(var + eps), of the unrounded x_new.
 * gate, scale, shift [seqs][cols], weight, post_weight [cols], each NULL for 1, 0, 0, 1 and no norm of
 * y; dtype is the rows', param_dtype the parameters': the same, or VMB_DTYPE_F32. y NULL: h alone is formed.
 * cols: a multiple of 8, at most 8192. Parameters and outputs are dense, 16-byte aligned.
 */
#define VMB_DTYPE_F32 2
typedef struct vmb_matrix {  /* [rows][cols], row stride in elements (a multiple of 8) */
  void* ptr;
  int64_t row;
} vmb_matrix;

typedef struct vmb_gated_norm_args {
  vmb_matrix x, y;                   /* y.ptr NULL: no block output */
  void *x_new, *h;                   /* forward outputs; x_new unused without y */
  const void *gate, *scale, *shift, *weight, *post_weight;
  float* stats;                      /* [3][rows]: written by the forward (NULL: not), read by the backward */
  const int32_t* seq_start;
  vmb_matrix dx_new, dh;             /* backward: gradients in, ptr NULL for zero */
  void *dx, *dy;                     /* backward outputs; dy unused without y */
  void *dgate, *dscale, *dshift, *dweight, *dpost_weight;  /* of param_dtype, each NULL if not wanted */
  int64_t rows;
  int32_t cols, seqs, dtype, param_dtype, layer;
  float eps;
  void* workspace; int64_t workspace_bytes;  /* backward, 256-byte aligned */
} vmb_gated_norm_args;

int64_t vmb_gated_norm_bwd_workspace_bytes(const vmb_gated_norm_args* a);  /* -1: malformed sizes */
int vmb_gated_norm_fwd(const vmb_gated_norm_args* a, void* stream);
int vmb_gated_norm_bwd(const vmb_gated_norm_args* a, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* VMONARCH_B200_H */
