/* libpots_mi355x — the C ABI of the MI355X verifier and commitment engine.
 *
 * Everything here runs on the current HIP device (gfx950). Pointers are plain addresses; a
 * "device" argument must be device memory of the current device, a "host" argument host
 * memory, and an argument documented as "host or device" may be either (the library asks HIP
 * which it is). Streams are passed as `void *` holding a hipStream_t (0 = the null stream).
 * No entry point throws; each returns a status (POTS_E_*) or a documented value, and
 * pots_last_error() describes the last HIP failure of the calling thread.
 *
 * The first group mirrors the reference's native batch (pacifai/pots-2.0,
 * verification/commitment/native.c) entry point by entry point, so the reference's ctypes
 * binding (verification/commitment/native.py:241-261) can load this library instead: the
 * names, argument order and meaning are the reference's, the hashing runs on the GPU, and
 * payloads and outputs may live in HBM. `n_threads` is accepted and ignored.
 */
#ifndef POTS_MI355X_H
#define POTS_MI355X_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define POTS_E_OK 0
#define POTS_E_NOMEM (-1)   /* the reference's "out of memory, nothing written" */
#define POTS_E_HIP (-3)     /* a HIP call failed; see pots_last_error() */
#define POTS_E_ARG (-4)     /* an argument is out of range or inconsistent */

/* Finiteness kinds (native.c:146-150): which payload values are tested for NaN/Inf. */
#define POTS_KIND_NONE 0
#define POTS_KIND_F32 1
#define POTS_KIND_BF16 2
#define POTS_KIND_F16 3

/* "pots-mi355x <version> gfx950". */
const char *pots_mi355x_version(void);

/* The last HIP error message of the calling thread, or "" if none. */
const char *pots_last_error(void);

/* Replaces native.c:341 pots_simd_degree: chunks compressed per instruction (64, one BLAKE3
 * chunk per lane of a wavefront). */
size_t pots_simd_degree(void);

/* Replaces native.c:343 pots_blake3_version: which BLAKE3 implementation hashes ("spec
 * (gfx950 kernels)": this library's own, written from the BLAKE3 specification). */
const char *pots_blake3_version(void);

/* ---- the reference's entry points --------------------------------------------------- */

/* Replaces native.c:243 pots_hash_leaves. Leaf i's digest BLAKE3(0x00 || header || payload)
 * goes to out + 32 i, the header being hdr_buf[hdr_off[u] : + hdr_len[u]] for u = hdr_idx[i]
 * and the payload payload_len[i] bytes at the address payload_ptr[i] (host or device memory).
 * kind[i] selects the NaN/Inf test (POTS_KIND_*). Metadata arrays and `out` are host memory.
 *
 * Returns the smallest i whose payload holds a non-finite value, or n when none does; the
 * digests before it are valid, those at or after it unspecified. Returns SIZE_MAX when a HIP
 * call fails (nothing valid written). Synchronous. */
size_t pots_hash_leaves(size_t n, const uint8_t *hdr_buf, const uint64_t *hdr_off,
                        const uint32_t *hdr_len, const uint32_t *hdr_idx,
                        const uint64_t *payload_ptr, const uint64_t *payload_len,
                        const uint8_t *kind, uint8_t *out, uint32_t n_threads);

/* No counterpart in the reference: pots_hash_leaves for callers that cannot allocate device
 * memory (code under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc). Same arguments, results and return values, bit for bit; it calls no hipMalloc,
 * hipFree or other allocating routine. Its workspace (the plan's descriptors and chaining
 * values, staged host payloads, the digests before their copy out) lives in a static 64 MiB
 * device array, one per GPU, held until the process ends: about 2 M chunks of 1 KiB, i.e.
 * some 2 GiB of leaf bytes in device memory (host payloads also take their size in it). A
 * larger request returns SIZE_MAX with the reason in pots_last_error(), before any GPU work.
 * The array belongs to the library's code object: loading the library reserves its 64 MiB
 * of device memory on each GPU where the code is loaded, even if this entry point is never
 * called.
 * Calls in one process are serialised, since they share the array; calls from two processes
 * on one GPU use separate arrays. Synchronous, on the null stream. */
size_t pots_hash_leaves_noalloc(size_t n, const uint8_t *hdr_buf, const uint64_t *hdr_off,
                                const uint32_t *hdr_len, const uint32_t *hdr_idx,
                                const uint64_t *payload_ptr, const uint64_t *payload_len,
                                const uint8_t *kind, uint8_t *out, uint32_t n_threads);

/* Replaces native.c:299 pots_all_finite: 1 when every value of the nbytes bytes at p (host
 * or device) is finite under `kind` (kind 0: always 1), 0 when one is NaN or Inf, a negative
 * POTS_E_* on failure. Synchronous. */
int pots_all_finite(const uint8_t *p, uint64_t nbytes, uint8_t kind, uint32_t n_threads);

/* Replaces native.c:335 pots_merkle_tree (which returns void): the 2n - 1 node hashes of the
 * RFC 6962 tree over n >= 1 leaf digests, pre-order (root first; for a range at p with left
 * half of k leaves, the left child at p + 1 and the right child at p + 2k), H_node(l, r) =
 * BLAKE3(0x01 || l || r). `leaves` (32 n bytes) and `nodes` (32 (2n - 1) bytes) are host or
 * device memory. Returns POTS_E_*. Synchronous. */
int pots_merkle_tree(size_t n, const uint8_t *leaves, uint8_t *nodes);

/* ---- stream-ordered entry points for a transcript resident in HBM ------------------- */

/* A leaf-hashing plan: the leaves' metadata uploaded once, the chunk decomposition and the
 * per-level reduction schedule computed, and the workspace allocated. Arguments as for
 * pots_hash_leaves, with every payload already in device memory (payload_ptr holds device
 * addresses; the arrays themselves are host memory). The caller keeps the payloads alive and
 * unmodified while runs of the plan are in flight. Returns POTS_E_*; *plan is set on success.
 * Replaces the batching of verification/commitment/leaves.py:312-437. */
int pots_leaf_plan_create(size_t n, const uint8_t *hdr_buf, const uint64_t *hdr_off,
                          const uint32_t *hdr_len, const uint32_t *hdr_idx,
                          const uint64_t *payload_ptr, const uint64_t *payload_len,
                          const uint8_t *kind, void **plan);

/* Enqueue the plan on `stream`: digests to d_out (device, 32 n bytes) and the smallest
 * non-finite leaf index (or n) to *d_first_bad (device uint32). No allocation, no sync. */
int pots_leaf_plan_run(void *plan, uint8_t *d_out, uint32_t *d_first_bad, void *stream);

/* pots_leaf_plan_run is these stages in order: 0 the staging copies and the first-bad reset,
 * 1 the chunk kernel (every 1 KiB chunk's chaining value, the NaN/Inf test fused), 2 the
 * per-leaf BLAKE3 trees above the chunks. Enqueued on `stream` one at a time, so a caller can
 * time each stage; the caller keeps the order. No counterpart in the reference. */
#define POTS_LEAF_STAGES 3
/* Stage 1 is two kernels, which a caller may also enqueue apart (each once, both before
 * stage 2): the chunks of the leaves fused with a Freivalds plan's products
 * (pots_leaf_plan_create_fused; it reads the challenges), and the chunks of the others. */
#define POTS_LEAF_STAGE_FUSED_CHUNKS 3
#define POTS_LEAF_STAGE_PLAIN_CHUNKS 4
int pots_leaf_plan_run_stage(void *plan, int stage, uint8_t *d_out, uint32_t *d_first_bad,
                             void *stream);

/* Limit the chunk kernels' grid to max_blocks blocks of 256 lanes (0: no limit, one block per
 * 256 slots; a slot is one lane's run of up to four consecutive chunks). Each block then
 * hashes several blocks' worth of slots in turn, and the kernel
 * holds at most that many blocks' worth of the GPU, leaving the rest to work on other
 * streams (the Freivalds passes, which are bound by HBM, not by the VALUs hashing needs).
 * Results do not depend on it. No counterpart in the reference. */
int pots_leaf_plan_set_grid(void *plan, uint32_t max_blocks);

/* As pots_leaf_plan_create, and the leaves that are the P operand of a product of fv_plan (a
 * Freivalds plan, below) also have that product's P-pass sums taken by the chunk kernel while
 * it hashes them, so P is read from HBM once for both checks. A product qualifies when the
 * plan's k is 1, 2 or 4, its P is the leaf's whole payload (contiguous, same dtype: bf16 or fp32, at a
 * 16-byte aligned address after a 12-byte 0x00 || header, i.e. a 2-D tensor leaf), its rows
 * hold at least 1 KiB, and no other product shares that P. The Freivalds plan's stage 4 then
 * reads what the chunk stage (stage 1 of this plan) wrote for the same claimed root: run
 * fv stage 0, then this plan's stage 1, before fv stage 4 (pots_step_run keeps that order on
 * one stream; pots_fv_plan_run refuses a fused plan). A Freivalds plan is fused with at most
 * one leaf plan; destroy the leaf plan first. Digests are those of pots_leaf_plan_create; the
 * rows agree with the unfused plan's to fp32 rounding of the sums' order. No counterpart in
 * the reference: it reads P once in check 2 and again in check 5. */
int pots_leaf_plan_create_fused(size_t n, const uint8_t *hdr_buf, const uint64_t *hdr_off,
                                const uint32_t *hdr_len, const uint32_t *hdr_idx,
                                const uint64_t *payload_ptr, const uint64_t *payload_len,
                                const uint8_t *kind, void *fv_plan, void **plan);

/* As pots_leaf_plan_create (fv_plan null) or pots_leaf_plan_create_fused, with the consecutive
 * chunks that a lane of the chunk kernels hashes given: run 1 to 4, or 0 for the plan's own
 * choice, which the other two take (by the number of chunks; few chunks take four lanes each, a
 * run given never does). Results do not depend on it. No counterpart in the reference. */
int pots_leaf_plan_create_runs(size_t n, const uint8_t *hdr_buf, const uint64_t *hdr_off,
                               const uint32_t *hdr_len, const uint32_t *hdr_idx,
                               const uint64_t *payload_ptr, const uint64_t *payload_len,
                               const uint8_t *kind, void *fv_plan, uint32_t run, void **plan);

/* Leaves of the plan whose product's P-pass sums its chunk stage takes (0 for an unfused
 * plan). */
uint32_t pots_leaf_plan_fused(const void *plan);

/* What one run of the fused chunk kernel moves: the fused leaves' message bytes (read), their
 * 1 KiB chunks (a 32-byte chaining value written each) and the run records it writes (32 bytes
 * each). Returns POTS_E_*. */
int pots_leaf_plan_fused_stats(const void *plan, uint64_t *msg_bytes, uint64_t *chunks,
                               uint64_t *records);

/* One step on one stream: fv stage 0, the leaf plan's stages, fv stages 1-5 (digests and
 * first-bad as pots_leaf_plan_run, rows as pots_fv_plan_run). For a fused pair of plans and
 * for two independent ones alike. No counterpart in the reference. */
int pots_step_run(void *leaf_plan, void *fv_plan, const uint8_t *d_key, uint8_t *d_digests,
                  uint32_t *d_first_bad, double *d_rows, void *stream);

/* Chunks (1 KiB BLAKE3 chunks) and message bytes the plan hashes. */
uint64_t pots_leaf_plan_chunks(const void *plan);
uint64_t pots_leaf_plan_bytes(const void *plan);

void pots_leaf_plan_destroy(void *plan);

/* The RFC 6962 tree over n leaf digests already in device memory, as pots_merkle_tree,
 * enqueued on `stream`; d_nodes (32 (2n - 1) bytes) is written in pre-order. */
int pots_merkle_tree_async(size_t n, const uint8_t *d_leaves, uint8_t *d_nodes, void *stream);

/* ---- Freivalds measurement and verdicts ---------------------------------------------- */

#define POTS_DT_F32 0
#define POTS_DT_BF16 1

/* One checked product P = A·B (+ 1·biasᵀ). All pointers are device memory; B and P are
 * row-major with the given row strides (elements). `bias` is fp32 [w] already rounded to the
 * operand format as the reference serves it (checks.py:439), or NULL. `m` is the product's
 * 1-based index, the challenge label.
 *
 * A is row-major with row stride lda when a_trans is 0. When a_trans is 1, A is the transpose
 * of a row-major X [q, n] at `a` with row stride lda, and another product of the same plan
 * must have that X as its row-major A (its twin: same pointer and lda, shape [q, n]); the
 * plan then reads X once for both (the twin pass). A transposed A is taken only in bf16, with
 * k <= 4, q a multiple of 16, n a multiple of 128, `a` and lda·2 multiples of 16 bytes;
 * anything else is POTS_E_ARG. No counterpart in the reference, which multiplies whatever
 * layout torch hands it. */
typedef struct {
  const void *a, *b, *p;
  const float *bias;
  uint64_t lda, ldb, ldp;
  uint32_t n, q, w, m;
  uint32_t a_dtype, b_dtype, p_dtype, a_trans;
} pots_fv_product;

/* A Freivalds plan over n products with k challenge vectors each: operand layout, column
 * chunking and workspace fixed once. Replaces the per-product torch op sequence of
 * verification/verifier/matmul_check/freivalds.py:290-321 and :384-410. guard = 0 leaves the
 * first two columns NaN (freivalds.py:309-312). */
int pots_fv_plan_create(size_t n, const pots_fv_product *products, uint32_t k, uint32_t guard,
                        void **plan);

/* Enqueue on `stream`: the 32 bytes at `key` (host memory, read before the call returns) to
 * d_key (device memory, 4-byte aligned), for the calls below that take a device-resident root.
 * No copy, no sync, no allocation. No counterpart in the reference. */
int pots_set_key_async(uint8_t *d_key, const uint8_t key[32], void *stream);

/* Enqueue on `stream`: the challenge matrices keyed on the 32-byte d_key (device memory,
 * the claimed root), the three streaming passes and the reduction, writing one fp64 row per
 * product to d_rows [n][5 + k] in freivalds.ROW order (freivalds.py:255): nu, ‖|P|1‖, ‖P‖_F,
 * Σ_i (A²(B²1))_i, ‖b‖², residual_1..k. No allocation, no sync. */
int pots_fv_plan_run(void *plan, const uint8_t *d_key, double *d_rows, void *stream);

/* pots_fv_plan_run keyed on 32 bytes of host memory (read before the call returns). */
int pots_fv_plan_run_root(void *plan, const uint8_t root[32], double *d_rows, void *stream);

/* pots_fv_plan_run is these stages in order: 0 the challenge matrices, 1 the B pass
 * (b1 = B·R, b2 = (B²)·1), 2 the reduction of B's split-K partials, 3 the A pass (A·b1 and
 * (A²)·b2), 4 the P pass (P·R, Σ|P|, ΣP²), 5 the rows. Enqueued on `stream` one at a time,
 * so a caller can time each stage; the caller keeps the order. No counterpart in the
 * reference. */
#define POTS_FV_STAGES 6
/* Stage 4 is two parts, which a caller may also enqueue apart (each once, both after stage 2
 * and before stage 5): the P pass over the products not fused with a leaf plan, and the fused
 * products' sums from the records the leaf plan's chunk stage wrote (nothing when unfused). */
#define POTS_FV_STAGE_P_PASS 6
#define POTS_FV_STAGE_P_FUSED 7
/* Stage 3 is two parts as well, which a caller may enqueue apart (each once, both after
 * stage 2 and before stage 5): the row pass over the A operands of products that have no
 * twin, and the twin pass over the twins' shared operands (nothing when the plan has none). */
#define POTS_FV_STAGE_A_ROWS 8
#define POTS_FV_STAGE_TWINS 9
int pots_fv_plan_run_stage(void *plan, int stage, const uint8_t *d_key, double *d_rows,
                           void *stream);

/* Limit the row-pass grid of stage 1 (B pass), 3 (A pass) or 4 (P pass) to max_blocks blocks
 * of 256 lanes (0: no limit, one block per tile). Each block then takes several tiles in turn,
 * from a queue per XCD (a contiguous range of the tiles each, then the other XCDs' ranges),
 * and the pass holds at most that many blocks' worth of the GPU, so that a kernel on another
 * stream (the leaf hasher, which needs every SIMD's VALUs) can share the CUs. Results do not
 * depend on it. No counterpart in the reference. */
int pots_fv_plan_set_grid(void *plan, int stage, uint32_t max_blocks);

/* Copy the last run's row-major challenge matrices (fp32; product i's [w_i, k] block follows
 * product i-1's) to d_out (device, Σ w_i·k floats), enqueued on `stream`. */
int pots_fv_plan_copy_challenges(const void *plan, float *d_out, void *stream);

/* Bytes of A, B and P the plan reads (each once). */
uint64_t pots_fv_plan_bytes(const void *plan);

/* The pairs of twin products the plan reads through the twin pass (a_trans products and their
 * row-major twins): each pair's shared operand is read once. No counterpart in the
 * reference. */
uint32_t pots_fv_plan_twins(const void *plan);

void pots_fv_plan_destroy(void *plan);

/* Replaces native.c:119 pots_challenges: item i's [widths[i], k] fp32 matrix at out +
 * offsets[i] (out host or device memory), vector j of product ms[i] the keyed XOF of
 * 0x10 || ms[i] (BE) || j under key, entries (2(w >> 8) + 1 - 2^24) / 2^24. Synchronous. */
int pots_challenges(const uint8_t key[32], uint32_t k, size_t n, const uint32_t *ms,
                    const uint32_t *widths, const uint64_t *offsets, float *out,
                    uint32_t n_threads);

/* Per-product verdicts from fp64 rows d_rows [n][5 + k] (device), on `stream`. d_specs is
 * device memory of n records { double kappa_max; uint32_t q, n, biased, pad; } (q the
 * checked contraction length, +1 with a bias). Writes (code, j) int32 pairs to d_codes
 * (0 accept, 1 non-finite, 2 cancellation guard, 3 residual of challenge j above tau·unit),
 * optionally (kappa, unit, U) to d_finished [n][3], and the smallest rejecting index (or n)
 * to *d_first_fail. sigma_r and sqrt2 are 1/√3 and √2 as the caller's doubles. Replaces
 * freivalds.py:324-335,450-468 and checks.py:926-956. */
int pots_verdicts_async(size_t n, const double *d_rows, uint32_t k, const void *d_specs,
                        double eps_in, double eps_acc, double tau, double sigma_r, double sqrt2,
                        uint32_t guard, uint32_t judge, int32_t *d_codes, double *d_finished,
                        uint32_t *d_first_fail, void *stream);

/* ---- check 6a: the SGD update identity of the linear weights ----------------------- */

/* One linear weight: W_t and W_{t+1} (fp32, n entries each) and the parts of its gradient G
 * (its committed weight-gradient products, fp32 or bf16, n entries each, summed in order in
 * fp32: chain_gradient, verification/computation/interface.py:169-180). All device memory,
 * contiguous. tau_w is the weight's band (bands.py tau_w_for). */
#define POTS_UPDATE_MAX_PARTS 8
typedef struct pots_update_weight {
  const void *w_t;
  const void *w_next;
  const void *parts[POTS_UPDATE_MAX_PARTS];
  uint32_t part_dtype[POTS_UPDATE_MAX_PARTS]; /* 0 fp32, 1 bf16 */
  uint32_t n_parts;
  uint32_t pad;
  uint64_t n;
  double tau_w;
} pots_update_weight;

/* Per weight, in device memory: rho_bits is ρ_max = max_i ρ_i as the bits of a double (NaN
 * if any ρ_i is NaN, 0 for an empty weight); first_nonfinite and first_over are the smallest
 * index whose R_i or scale_i is not finite, and whose ρ_i is not ≤ tau_w, or UINT64_MAX. */
typedef struct pots_update_result {
  uint64_t rho_bits;
  uint64_t first_nonfinite;
  uint64_t first_over;
} pots_update_result;

/* A plan over n weights, with the step size eta and ε_W (eps_w) already rounded to fp32 (the
 * reference multiplies fp32 tensors by them as fp32 scalars). Replaces the per-weight work of
 * checks.py:380-451 (_update_identity, _update_identity_reference; ρ_max bit for bit as
 * _fast_rho_max, checks.py:301-377, obtains it): R = |W_{t+1} − (W_t − η·G)|,
 * scale = ε_W·(|W_t| + |η·G|) in fp32, ρ_i = 0 if R_i = 0 else fl64(R_i)/fl64(scale_i). */
int pots_update_plan_create(size_t n, const pots_update_weight *weights, float eta, float eps_w,
                            void **plan);
/* Enqueue the pass; d_out holds n results (device). Stream-ordered, no allocation, no sync. */
int pots_update_plan_run(void *plan, pots_update_result *d_out, void *stream);
/* Bytes one run reads: W_t, W_{t+1} and every gradient part once. */
uint64_t pots_update_plan_bytes(void *plan);
void pots_update_plan_destroy(void *plan);

/* ---- Stored steps: leaf files to device memory ------------------------------------------
 *
 * The on-disk transcript store (verification/transcript/store.py:285-380, DiskStore) writes
 * one torch.save file per leaf. Its reader (store.py:347-357, DiskStore.leaf) unpickles each
 * file into pageable host memory with torch.load; the checks then copy the tensors to the GPU
 * one by one. These two entry points replace that read for a whole step: a parallel scan of
 * the files' ZIP directories and pickles (no Python, nothing executed), then parallel reads
 * of the storage bytes into pinned staging and DMA into one device buffer. */

#define POTS_E_IO (-5) /* a file could not be opened or read; see pots_last_error() */

/* Element types of a stored tensor, from its pickled storage class (torch.FloatStorage ...). */
#define POTS_STORE_F32 1
#define POTS_STORE_F64 2
#define POTS_STORE_F16 3
#define POTS_STORE_BF16 4
#define POTS_STORE_I64 5
#define POTS_STORE_I32 6
#define POTS_STORE_I16 7
#define POTS_STORE_I8 8
#define POTS_STORE_U8 9
#define POTS_STORE_BOOL 10

/* Scan status of one file. */
#define POTS_STORE_OK 0     /* one plain tensor, described below */
#define POTS_STORE_OTHER 1  /* anything else (a record's dict, a tensor that needs grad, a
                               big-endian or compressed archive, ...): read it with torch.load */
#define POTS_STORE_UNREADABLE 2 /* not a ZIP archive that can be read; torch.load fails too */

#define POTS_STORE_MAX_DIM 8

/* What pots_store_scan found in one file: a tensor of `ndim` dims with these sizes and
 * strides (elements) at `storage_offset` elements into a storage of `storage_bytes` bytes,
 * stored uncompressed at `data_offset` in the file. Fields other than status are meaningful
 * only for POTS_STORE_OK. */
typedef struct pots_stored_tensor {
  uint64_t data_offset;
  uint64_t storage_bytes;
  uint64_t storage_offset;
  int64_t size[POTS_STORE_MAX_DIM];
  int64_t stride[POTS_STORE_MAX_DIM];
  uint32_t ndim;
  uint32_t dtype; /* POTS_STORE_F32 ... */
  int32_t status; /* POTS_STORE_OK ... */
  uint32_t pad;
} pots_stored_tensor;

/* Scan n_files files on n_threads host threads (0: 8). Accepts exactly the pickle torch.save
 * writes for one tensor that does not require grad, torch._utils._rebuild_tensor_v2(storage,
 * offset, size, stride, False, OrderedDict()), with a little-endian byte order record and the
 * storage's record stored; its opcodes are walked, never executed. Returns POTS_E_OK (each
 * file's own outcome is in its status) or POTS_E_ARG. Host only: needs no GPU. */
int pots_store_scan(uint32_t n_files, const char *const *paths, pots_stored_tensor *out,
                    uint32_t n_threads);

/* One piece of a file for pots_store_load: `bytes` bytes at `file_offset` of file `file` go
 * to `dst_offset` bytes into the destination. */
typedef struct pots_store_segment {
  uint32_t file;
  uint32_t pad;
  uint64_t file_offset;
  uint64_t bytes;
  uint64_t dst_offset;
} pots_store_segment;

/* Copy the segments (sorted by dst_offset, not overlapping) into `dst`. With dst_device >= 0,
 * dst is memory of that device: n_threads host threads (0: 8) each read their share of the
 * spans into two slots of the pinned host `staging` (staging_bytes, at least 2·n_threads·64
 * KiB, from hipHostMalloc) and send each slot with one hipMemcpyAsync on a stream of their
 * own. With dst_device < 0, dst is host memory read into directly (staging unused). Bytes
 * between segments that fall inside one span are written with unspecified values. Returns
 * after every copy has completed: POTS_E_OK, POTS_E_IO (a short or failed read), POTS_E_HIP
 * or POTS_E_ARG. */
int pots_store_load(uint32_t n_files, const char *const *paths, uint32_t n_segs,
                    const pots_store_segment *segs, void *dst, int dst_device, void *staging,
                    uint64_t staging_bytes, uint32_t n_threads);

/* ---- The training pass's own operators ---------------------------------------------------
 *
 * Attention, the loss over a vocabulary and the embedding, each with its gradient, for a pass
 * that is not captured: no attention probability and no logit is kept. Every pointer is device
 * memory of the current device; the calls enqueue on `stream` and allocate nothing; `work` is
 * scratch of at least the size the matching *_work call returns, aligned to 256 bytes, its
 * contents neither read before nor kept after a call. Results do not depend on the order in
 * which blocks run. They return POTS_E_OK, POTS_E_ARG (a size, type or stride out of range; no
 * work enqueued) or POTS_E_HIP. */

#define POTS_OP_F32 0
#define POTS_OP_BF16 1

#define POTS_ATTENTION_MAX_DIM 128

/* One operand [batch, heads, n, head_dim]: elements between batches, heads and positions (a
 * position's values are consecutive). The pointer and every stride are multiples of 16 bytes, and
 * `row` is less than 2^22. */
typedef struct pots_heads {
  void *ptr;
  int64_t batch, head, row;
} pots_heads;

/* Softmax attention of `batch` sequences of n positions over their own keys: `heads` query
 * heads, each `heads / kv_heads` consecutive ones sharing a key head, of a head_dim that is a
 * multiple of 8 (a narrower head is one with columns of zeros); batch * heads is at most 2^20,
 * and there are less than 2^24 blocks of 128 rows of all heads (half of that backward for heads
 * wider than 64). Position i sees j where j < length, i < length and (causal) j <= i; lengths is
 * int32 [batch] (values past n count as n, negative ones as 0), or null for n. A position that
 * sees nothing has an output of zero, lse -inf and gradients of zero; what lies past a sequence's
 * length is not read. lse is fp32 [batch, heads, n], natural logarithms. */
typedef struct pots_attention {
  pots_heads q, k, v, out;
  pots_heads dout, dq, dk, dv; /* backward only */
  float *lse;                  /* forward: written; backward: read */
  const int32_t *lengths;
  uint32_t batch, heads, kv_heads, n, head_dim;
  uint32_t dtype, causal;
  float scale;
} pots_attention;

int pots_attention_forward(const pots_attention *a, void *stream);
uint64_t pots_attention_backward_work(const pots_attention *a);
int pots_attention_backward(const pots_attention *a, void *work, void *stream);

/* Softmax cross entropy of feature rows x [rows, dim] against a vocabulary matrix w
 * [vocab, dim]: loss_r = lse_r - x_r.w_t, fp32, with t the row's int64 target; 0 where t < 0, NaN
 * where t >= vocab. Backward: dx and dw of sum_r weights_r loss_r; a row of weight zero or without a
 * target counts for nothing, whatever its features. Rows of x, w, dx and dw are `*_row`
 * elements apart. Up to 2^24 rows and vocabulary entries and 2^16 columns. */
typedef struct pots_vocab_loss {
  const void *x, *w;
  const int64_t *targets;
  float *loss, *lse;    /* [rows]; forward: both written; backward: lse is read */
  const float *weights; /* [rows], backward only */
  void *dx, *dw;        /* backward only */
  int64_t x_row, w_row, dx_row, dw_row;
  uint32_t rows, dim, vocab, dtype;
} pots_vocab_loss;

uint64_t pots_vocab_loss_forward_work(const pots_vocab_loss *a);
int pots_vocab_loss_forward(const pots_vocab_loss *a, void *work, void *stream);
uint64_t pots_vocab_loss_backward_work(const pots_vocab_loss *a);
int pots_vocab_loss_backward(const pots_vocab_loss *a, void *work, void *stream);

/* Rows of a table [vocab, dim] by token, times scale: out_i = scale * table[ids_i] (NaN where
 * ids_i is outside the table). Backward: table_v (+)= scale * the sum of rows_i over ids_i = v, in
 * fp32, added up in runs of consecutive i and the runs in order; with `add` it is added to what the
 * table holds, without it every row is written. An id outside the table adds to nothing. Up to 2^24
 * tokens, 2^30 rows and 2^20 columns. */
typedef struct pots_embedding {
  const int64_t *ids;
  void *table;
  void *rows; /* forward: written; backward: read */
  int64_t table_row, rows_row;
  uint32_t tokens, dim, vocab, dtype;
  uint32_t add;
  float scale;
} pots_embedding;

int pots_embedding_forward(const pots_embedding *a, void *stream);
uint64_t pots_embedding_backward_work(const pots_embedding *a);
int pots_embedding_backward(const pots_embedding *a, void *work, void *stream);

/* ---- What a training step does between its products, and after them -----------------------
 *
 * The residual's addition with the root-mean-square norm, rotary turns of queries and keys, the
 * gated activation, and the clipped update of the weights; as above: device memory, calls that
 * enqueue and allocate nothing, `work` of the *_work call's size, results that do not depend on
 * the order of blocks. Rows start anywhere that an element may: `*_row` elements apart, the values
 * of a row consecutive. */

#define POTS_OP_E4M3 2 /* outputs of pots_rms_norm_quantized alone */
#define POTS_OP_INT8 3
#define POTS_OP_F64 4 /* the frequencies of pots_rotary alone */

/* t = x + residual (rounded to total_type; x itself where residual is null, and total is then not
 * written); s = 1 / sqrt(mean of t^2 over the row + eps), eps at least 2^-126; y = t s weight. rstd receives s; the
 * rows of y and total follow each other. Up to 2^14 columns and 2^31 - 1 rows.
 * Quantized: y / scale in e4m3 or int8, to nearest (ties to even), with a scale for each `block`
 * columns (32, 64, 128 or 256; 0: the whole row): the largest size of y there over 448 or 127, at
 * least 2^-126. Where y holds a NaN the block's scale is NaN; where it holds an infinity the scale is
 * infinite, and what is finite in the block 0. y / scale is NaN of the whole block with a NaN scale and of the infinities: a
 * NaN in e4m3, -128 in int8, whose numbers else are -127 to 127.
 * Backward, h = t s and g = dy weight: dt = dtotal + s (g - h mean(g h)), to dresidual in
 * total_type and to dx in x_type (each may be null, and so may dtotal), their rows following each
 * other; dweight (may be null) is the rows' sum of dy h, in weight_type. x, residual and y are not
 * read. */
typedef struct pots_rms_norm {
  const void *x, *residual, *weight;
  void *total; /* forward: written; backward: read */
  void *y;
  float *rstd;   /* [rows]; forward: written; backward: read */
  float *scales; /* [rows][blocks], quantized only */
  const void *dy, *dtotal;
  void *dx, *dresidual, *dweight;
  int64_t x_row, residual_row, total_row, dy_row, dtotal_row; /* total_row: backward only */
  uint32_t rows, dim, block;
  uint32_t x_type, total_type, weight_type, y_type; /* y_type: of y and dy */
  float eps;
} pots_rms_norm;

int pots_rms_norm_forward(const pots_rms_norm *a, void *stream);
int pots_rms_norm_quantized(const pots_rms_norm *a, void *stream);
uint64_t pots_rms_norm_backward_work(const pots_rms_norm *a);
int pots_rms_norm_backward(const pots_rms_norm *a, void *work, void *stream);

/* Pairs (u, v) of each head of q [batch, heads, n, head_dim] and k [batch, kv_heads, ...], turned to
 * (u cos - v sin, u sin + v cos) by the angle position * frequency of the pair (`inverse`: by its
 * negative, which is the gradient). Pair i is (i, i + pairs), or (2i, 2i + 1) where `adjacent`;
 * columns from 2 * pairs on are copied. Its position is that of the axis a with
 * ends[a - 1] <= i < ends[a]: int32 or int64 at positions + a * position_axis + batch *
 * position_batch + token * position_token (elements). Angles are taken in 64 bits. Strides and
 * pointers of heads are any that an element may have. Up to 2^10 columns, 4 axes, 2^31 - 1 tokens and
 * 2^16 heads. q_out and k_out are not the inputs' memory. */
typedef struct pots_rotary {
  pots_heads q, k, q_out, k_out;
  const void *positions, *frequencies;
  int64_t position_axis, position_batch, position_token;
  uint32_t batch, heads, kv_heads, n, head_dim, pairs, axes;
  uint32_t ends[4];
  uint32_t dtype, frequency_type, position_bits; /* frequencies: POTS_OP_F32 or POTS_OP_F64 */
  uint32_t adjacent, inverse;
} pots_rotary;

int pots_rotary_turn(const pots_rotary *a, void *stream);

/* out = silu(gate) * up, silu(g) = g / (1 + e^-g); backward: dgate and dup of it. The rows of out,
 * dgate and dup follow each other. rows * columns is at most 2^40; any count of columns. */
typedef struct pots_gated_silu {
  const void *gate, *up, *dout;
  void *out, *dgate, *dup;
  int64_t gate_row, up_row, dout_row;
  uint32_t rows, columns, dtype;
} pots_gated_silu;

int pots_gated_silu_forward(const pots_gated_silu *a, void *stream);
int pots_gated_silu_backward(const pots_gated_silu *a, void *stream);

/* The 2-norm of many tensors' values together, from a sum of squares in 64 bits, to norm; and with
 * factor = max_norm / norm where the norm exceeds max_norm and 1 elsewhere (a NaN norm has a NaN
 * factor; an infinite max_norm is no bound, and the factor is 1 whatever the norm): clip, out = factor * gradient in gradient_type; step, out = weight - eta * factor *
 * gradient in weight_type. The `tensors` entries (1 to 2^16) follow the block in memory. Values of a
 * tensor are consecutive, from where an element may start. An out may be its own gradient or
 * weight; two outs that overlap, or an out over another input or shifted over its own, are refused. */
typedef struct pots_gradients {
  float *norm;
  float max_norm, eta;
  uint32_t tensors, pad;
} pots_gradients;

typedef struct pots_gradient {
  const void *gradient, *weight; /* weight: step only */
  void *out;
  uint64_t count;
  uint32_t gradient_type, weight_type;
} pots_gradient;

uint64_t pots_gradient_norm_work(const pots_gradients *a);
int pots_gradient_norm(const pots_gradients *a, void *work, void *stream);
uint64_t pots_clip_gradients_work(const pots_gradients *a);
int pots_clip_gradients(const pots_gradients *a, void *work, void *stream);
uint64_t pots_sgd_step_work(const pots_gradients *a);
int pots_sgd_step(const pots_gradients *a, void *work, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* POTS_MI355X_H */
