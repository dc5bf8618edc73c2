/*
 * omeinsum_b200.h -- C ABI of the B200 (sm_100a) execution backend for
 * omeinsum-rs.
 *
 * The entry points replace the reference's `Backend` trait for a new `B200`
 * backend (tensor4all/omeinsum-rs, src/backend/traits.rs:42-199): a Rust
 * `impl Backend for B200` binds them one-to-one.
 *
 * Conventions (same as the reference):
 *   - tensors are column-major: axis 0 is fastest; strides count ELEMENTS;
 *   - modes are arbitrary int32 labels, unique within one operand;
 *   - a mode in A, B and C is a batch mode; in A and B only, contracted; in
 *     one input and C, free; in one input only, traced (reduced first);
 *   - outputs are written contiguous column-major in modes_c order;
 *   - argmax (u32) is the column-major linear index over the contracted
 *     modes, taken in modes_a order; ties go to the smallest index;
 *   - MaxPlus zero = -FLT_MAX (f32::MIN), MinPlus zero = +FLT_MAX, MaxMul zero = 0.
 *
 * All device pointers are plain CUDA device addresses on the backend's device.
 * Every call is ordered on the backend's own stream; om_b200_sync waits for it.
 * Every function returns OM_OK (0) or an OM_ERR_* code; om_b200_last_error
 * gives the message of the last failure on the calling thread.
 */
#ifndef OMEINSUM_B200_H
#define OMEINSUM_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct om_backend om_backend;

/* semirings: src/algebra/standard.rs, src/algebra/tropical.rs */
typedef enum {
  OM_STANDARD = 0, /* (+, x)   zero 0            */
  OM_MAXPLUS = 1,  /* (max, +) zero -FLT_MAX     */
  OM_MINPLUS = 2,  /* (min, +) zero +FLT_MAX     */
  OM_MAXMUL = 3    /* (max, x) zero 0            */
} om_algebra;

/* OM_C32 / OM_C64: complex numbers as interleaved (re, im) pairs of
 * f32 / f64 (the layout of num_complex::Complex and of the reference's
 * CudaComplex, src/backend/cuda/mod.rs:56-208); Standard algebra only. */
typedef enum {
  OM_F32 = 0,
  OM_F64 = 1,
  OM_U32 = 2,
  OM_C32 = 3,
  OM_C64 = 4,
  /* taken by the sequence-model operators only (end of this header) */
  OM_BF16 = 5,
  OM_F16 = 6,
  OM_I8 = 7,
  OM_I32 = 8,
  OM_I64 = 9
} om_dtype;

enum {
  OM_OK = 0,
  OM_ERR_INVALID = 1,     /* bad argument: null pointer, bad rank, size mismatch */
  OM_ERR_UNSUPPORTED = 2, /* dtype / algebra combination not provided            */
  OM_ERR_CUDA = 3,        /* CUDA runtime error                                  */
  OM_ERR_OOM = 4,         /* device allocation failed                            */
  OM_ERR_SHAPE = 5,       /* modes / shapes inconsistent                         */
  OM_ERR_NCCL = 6,        /* collective failed                                   */
  OM_ERR_TIMEOUT = 7      /* a bounded wait ran out                              */
};

#define OM_MAX_DIMS 64

/* Backend::name (traits.rs:50) -- returns "b200". */
const char* om_b200_name(void);

/* Copies the last error message of this thread into buf (NUL-terminated). */
int om_b200_last_error(char* buf, size_t len);

/* Creates a backend bound to CUDA device `device` with its own non-blocking
 * stream and a stream-ordered caching allocator.  Mirrors `Cuda::on_device`
 * (src/backend/cuda/mod.rs:258-265): a bad ordinal is an error, not a panic. */
int om_b200_create(int device, om_backend** out);
int om_b200_destroy(om_backend* be);

/* A backend whose work is ordered on the caller's stream (a cudaStream_t of
 * `device`; NULL = the legacy default stream) instead of one of its own, for
 * hosts that keep their tensors on a stream already.  The stream is borrowed:
 * it must outlive the backend and om_b200_destroy leaves it open.  No
 * counterpart in the reference.  Recording (om_b200_graph_begin) needs a
 * stream that can be captured, so not the legacy default stream. */
int om_b200_create_on_stream(int device, void* stream, om_backend** out);

/* The backend's stream (a cudaStream_t), for callers that interoperate. */
int om_b200_stream(om_backend* be, void** stream_out);

/* Backend::synchronize (traits.rs:53). */
int om_b200_sync(om_backend* be);

/* Backend::alloc (traits.rs:56): zero-filled device buffer of `bytes`. */
int om_b200_alloc(om_backend* be, size_t bytes, void** dptr);
int om_b200_free(om_backend* be, void* dptr);

/* Backend::from_slice (traits.rs:60) is alloc + upload; Storage::to_vec
 * (traits.rs:20) is download.  Both are stream-ordered; download waits. */
int om_b200_upload(om_backend* be, void* dst_device, const void* src_host, size_t bytes);
int om_b200_download(om_backend* be, void* dst_host, const void* src_device, size_t bytes);
/* om_b200_download without the wait: the copy is queued on the backend's
 * stream and dst_host must stay valid until om_b200_sync returns (use pinned
 * host memory for a truly asynchronous copy).  No counterpart in the
 * reference (Storage::to_vec always waits); a caller that overlaps one
 * step's copies with another step's contraction on a second backend uses it. */
int om_b200_download_async(om_backend* be, void* dst_host, const void* src_device, size_t bytes);

/* Backend::copy_strided (traits.rs:71-77): gathers the strided view
 * (shape, strides, offset in elements) of src into the contiguous
 * column-major dst.  dtype gives the element size (OM_U32 allowed). */
int om_b200_copy_strided(om_backend* be, om_dtype dtype, const void* src, int ndim,
                         const int64_t* shape, const int64_t* strides, int64_t offset, void* dst);

/* Backend::contract (traits.rs:147-166) when argmax_out == NULL, and
 * Backend::contract_with_argmax (traits.rs:180-199) otherwise.  The output
 * c_out (and argmax_out) hold prod(shape_c) elements (1 when ndc == 0).
 * Inputs are read through their strides; nothing is copied back to the host. */
int om_b200_contract(om_backend* be, om_algebra alg, om_dtype dtype,
                     const void* a, int nda, const int64_t* shape_a, const int64_t* strides_a,
                     const int32_t* modes_a,
                     const void* b, int ndb, const int64_t* shape_b, const int64_t* strides_b,
                     const int32_t* modes_b,
                     int ndc, const int64_t* shape_c, const int32_t* modes_c,
                     void* c_out, uint32_t* argmax_out);

/* Unary einsum ix -> iy (execute_unary_naive / execute_unary_with_argmax,
 * src/einsum/engine.rs:752-926): trace, diagonal, reduction, permutation and
 * diagonal embedding.  ix may repeat labels; iy may repeat labels (off-diagonal
 * entries get the algebra's zero).  sizes_y[d] is the size of iy[d]; the input
 * is read through shape_x/strides_x.  argmax_out (optional) receives the
 * column-major linear input position of the winner (is_better, first wins). */
int om_b200_unary(om_backend* be, om_algebra alg, om_dtype dtype,
                  const void* x, int nx, const int32_t* ix, const int64_t* shape_x,
                  const int64_t* strides_x,
                  int ny, const int32_t* iy, const int64_t* sizes_y,
                  void* y_out, uint32_t* argmax_out);

/* Tropical backward of one binary node (src/einsum/backward.rs:90-166):
 * scatters grad_c into grad_a / grad_b (contiguous, column-major, shapes of
 * the normalised operands, ACCUMULATED into) through the argmax of the
 * forward contraction.  Operands are given by shape and modes only. */
int om_b200_tropical_backward(om_backend* be, om_dtype dtype,
                              const void* grad_c, const uint32_t* argmax,
                              int nda, const int64_t* shape_a, const int32_t* modes_a,
                              int ndb, const int64_t* shape_b, const int32_t* modes_b,
                              int ndc, const int64_t* shape_c, const int32_t* modes_c,
                              void* grad_a, void* grad_b);

/* Arithmetic of Standard<f32> products (no counterpart in the reference,
 * whose faer path is plain f32):
 *   OM_F32_TENSOR_3XTF32 (default): shapes of at least 64 x 64 x 16 run on the
 *     tensor cores (tcgen05) as three TF32 products per f32 product
 *     (A_lo B_hi + A_hi B_lo + A_hi B_hi) accumulated in f32; the error is
 *     about 2^-21 * sum_k |a||b|.  Smaller shapes use the exact path.
 *   OM_F32_EXACT: every Standard f32 product is an f32 FMA on the CUDA cores.
 * The environment variable OM_DISABLE_TCGEN05 (any value) makes OM_F32_EXACT
 * the default of new backends.  f64 and the tropical algebras are unaffected. */
typedef enum { OM_F32_TENSOR_3XTF32 = 0, OM_F32_EXACT = 1 } om_f32_mode;
int om_b200_set_f32_mode(om_backend* be, om_f32_mode mode);

/* dst[idx[i]] = src[i] (accumulate == 0) or dst[idx[i]] += src[i]
 * (accumulate != 0) for 0 <= i < n; idx is a device array of distinct int64
 * element offsets into dst.  No counterpart in the reference: the sliced
 * network driver uses it to place a slice's gradients (views of the inputs)
 * into the full gradient tensors on the device, and to sum slices there. */
int om_b200_scatter_index(om_backend* be, om_dtype dtype, const void* src, int64_t n,
                          const int64_t* idx, void* dst, int accumulate);

/* Many strided gathers in one launch (no counterpart in the reference: the
 * sliced network driver stages a slice's views of the sliced input tensors
 * with it).  desc (device) holds nviews descriptors of 28 int64 words each:
 * source pointer, destination pointer, ndim (<= 12), element count, then 12
 * extents and 12 element strides (column-major odometer over the extents).
 * View v of slice s starts at element offsets[s * nviews + v] (device) of its
 * source; s is read on the device from *sel, so a graph recorded around this
 * call serves every slice.  Destinations are contiguous.  max_numel bounds
 * the views' element counts (it sizes the grid). */
int om_b200_gather_views(om_backend* be, om_dtype dtype, int nviews, const int64_t* desc,
                         const int64_t* offsets, const int32_t* sel, int64_t max_numel);

/* Contraction-order optimisation by tree simulated annealing (host code;
 * replaces the reference's call into omeco's optimize_treesa,
 * src/einsum/engine.rs:84-91).  Network as in om_b200_einsum (ntensors,
 * ndims, ixs, iy, size dictionary).  init_children (2 * (ntensors - 1),
 * post order, may be NULL) seeds the first of ntrials runs; the others start
 * from random trees.  Cost: log2 sum of 2^tc over nodes + sc_weight * sum
 * of max(0, log2 size - sc_target) over intermediates + rw_weight * log2 of
 * the read-write volume; Metropolis moves (rotations at a node), beta from
 * beta_start to beta_end by beta_step, niters sweeps per beta.  Writes the
 * best tree to children_out (post order) and its log2 time / space
 * complexity to tc_out / sc_out (may be NULL). */
int om_b200_optimize_tree(int ntensors, const int32_t* ndims, const int32_t* ixs, int niy,
                          const int32_t* iy, int nsizes, const int32_t* size_labels,
                          const int64_t* size_values, const int32_t* init_children,
                          double sc_target, double sc_weight, double rw_weight, int ntrials,
                          int niters, double beta_start, double beta_end, double beta_step,
                          uint64_t seed, int32_t* children_out, double* tc_out, double* sc_out);

/* Kernel launches issued by this thread since the last call (counter reset
 * on read); used by benchmarks to report how many device kernels ran. */
int64_t om_b200_launch_count(void);

/* Per-kernel device timing: with profiling on, each kernel launch of this
 * backend is bracketed by CUDA events on the backend's stream.  Turning it on
 * clears the accumulators.  om_b200_profile_query synchronises the stream and
 * returns, for kernel class `index` (0, 1, ...), its name, summed device time
 * and launch count; OM_ERR_INVALID once index runs past the last class. */
int om_b200_profile_enable(om_backend* be, int on);
int om_b200_profile_query(om_backend* be, int index, char* name, size_t len, double* total_ms,
                          int64_t* launches);

/* ---- einsum engine over a contraction tree --------------------------------
 * Restates Einsum::execute / execute_with_argmax and the gradient tape of
 * cost_and_gradient (src/einsum/engine.rs:125-301,392-578;
 * src/einsum/backward.rs:405-799) on the device.
 *
 * Inputs: `ntensors` device tensors; tensor t has rank ndims[t], and its
 * shape, strides and labels are the next ndims[t] entries of shapes / strides
 * / ixs (concatenated over t).  Labels are int32 >= 0; size_labels[q] has
 * extent size_values[q] (the size dictionary).  iy (length niy) are the
 * output labels.
 *
 * Tree: `nnodes` binary nodes in post order.  Node i contracts children
 * children[2i], children[2i+1]; a child value c < ntensors is leaf tensor c,
 * c >= ntensors is node c - ntensors.  Its output labels are
 * node_iy[node_iy_off[i] .. node_iy_off[i+1]).  The last node is the root.
 * nnodes == 0 means the tree is the single leaf 0 (a unary einsum).
 *
 * Operands are normalised before each node (labels in neither the other
 * operand nor the node output are reduced first, repeated labels take the
 * diagonal), and the root is reduced / permuted to iy at the end.  `out`
 * receives prod(extent of iy) contiguous column-major elements.
 *
 * With tape_out non-NULL the forward keeps a gradient tape (argmax of every
 * node for the tropical algebras, every intermediate for Standard); pass it
 * to om_b200_einsum_backward, then free it with om_b200_tape_free. */
typedef struct om_tape om_tape;
int om_b200_einsum(om_backend* be, om_algebra alg, om_dtype dtype, int ntensors,
                   const void* const* tensors, const int32_t* ndims, const int64_t* shapes,
                   const int64_t* strides, const int32_t* ixs, int niy, const int32_t* iy,
                   int nsizes, const int32_t* size_labels, const int64_t* size_values,
                   int nnodes, const int32_t* children, const int32_t* node_iy_off,
                   const int32_t* node_iy, void* out, om_tape** tape_out);

/* om_b200_einsum with a tape of values only (tropical algebras): every
 * intermediate is kept, but no node computes its argmax.  The backward
 * (om_b200_einsum_backward / _linked, outputs of at most 4096 elements)
 * then finds the argmax of just the elements the gradient visits, from the
 * children's values, with the same rule as the forward (generic_gemm_with_argmax,
 * src/backend/cpu/mod.rs:889-920, and execute_unary_with_argmax,
 * src/einsum/engine.rs:841-926), so the gradient is the one the argmax tape
 * gives.  No counterpart in the reference: it lets a caller contract many
 * candidates (the slices of a sliced network) at value cost and take the
 * gradient of the winner only. */
int om_b200_einsum_tape_values(om_backend* be, om_algebra alg, om_dtype dtype, int ntensors,
                               const void* const* tensors, const int32_t* ndims,
                               const int64_t* shapes, const int64_t* strides, const int32_t* ixs,
                               int niy, const int32_t* iy, int nsizes, const int32_t* size_labels,
                               const int64_t* size_values, int nnodes, const int32_t* children,
                               const int32_t* node_iy_off, const int32_t* node_iy, void* out,
                               om_tape** tape_out);

/* GradientTape::backward (backward.rs:498-506, 678-728): given dy (shaped
 * like the output, contiguous), writes the gradient of every input tensor t,
 * contiguous column-major in the input's shape, to grads[t]. */
int om_b200_einsum_backward(om_tape* tape, const void* dy, void* const* grads);

/* One backward through several tapes (no counterpart in the reference):
 * input tensor link_leaf[i] of `tape` is the output of the contraction
 * recorded in link_tapes[i] (same algebra and dtype, its output contiguous in
 * that leaf's label order); the gradient continues through it, and the
 * inputs of link_tapes[i] receive theirs in link_grads[i][...].  grads[] of
 * linked leaves are not written.  Tropical tapes whose output has at most
 * 4096 elements only (the walk of om_b200_einsum_backward for small
 * gradients, in one launch for all tapes); otherwise OM_ERR_UNSUPPORTED. */
int om_b200_einsum_backward_linked(om_tape* tape, const void* dy, void* const* grads, int nlinks,
                                   const int32_t* link_leaf, om_tape* const* link_tapes,
                                   void* const* const* link_grads);
int om_b200_tape_free(om_tape* tape);

/* For a tape recorded inside a graph (om_b200_graph_begin/end): frees the
 * device buffers the tape refers to, stream-ordered, and keeps the tape.  A
 * later replay of the graph allocates the same addresses again, after which
 * om_b200_einsum_backward may run on the tape once more.  This keeps a
 * recorded tape from holding its memory between replays.  Not meant for
 * tapes made outside a graph (their buffers would not come back). */
int om_b200_tape_release(om_tape* tape);

/* Stream capture into a CUDA graph.  No counterpart in the reference (its
 * CPU backend has no launch cost to amortise); it serves callers that repeat
 * the same sequence of library calls on the same buffers, such as the slices
 * of a sliced network.  Between om_b200_graph_begin and om_b200_graph_end,
 * work issued on the backend's stream (om_b200_contract, om_b200_einsum,
 * copies, ...) is recorded instead of run; the library's own stream-ordered
 * allocations inside become part of the graph.  om_b200_graph_launch runs the
 * recorded work on the backend's stream.  Calls that wait for the device
 * (om_b200_sync, om_b200_download, profile queries) must not be made while
 * capturing. */
typedef struct om_graph om_graph;
int om_b200_graph_begin(om_backend* be);
int om_b200_graph_end(om_backend* be, om_graph** graph_out);
int om_b200_graph_launch(om_backend* be, om_graph* graph);
int om_b200_graph_free(om_graph* graph);

/* Concurrent branches of a recording (no reference counterpart): after
 * om_b200_graph_branch(be, b) with 0 <= b < 64, the work issued on the
 * backend is recorded on branch b, which starts after everything recorded
 * before the first branch call; om_b200_graph_branch(be, -1) returns to the
 * backend's own stream.  om_b200_graph_end joins every branch, so the graph
 * ends after all of them.  Branches run concurrently at replay and must use
 * disjoint buffers; blocks the library frees inside them are not reused
 * within the recording.  Tropical f32 GEMMs inside branches take the exact
 * compare-select path (the fast path's gate word is one per backend). */
int om_b200_graph_branch(om_backend* be, int branch);

/* Allocation-free tropical matrix product with argmax.  No counterpart in the
 * reference: it exists for callers that must not allocate device memory
 * while they run (a host that hands all device memory out of its own arena,
 * a latency-critical path where an allocation could block or fail, an
 * embedder that forbids library-owned allocations).
 *
 * C = A (x) B in MaxPlus / MinPlus / MaxMul f32, with the u32 argmax of the
 * first winning k (same results as om_b200_contract with modes
 * 'ij,jk->ik').  A (m x k, leading dimension lda), B (k x n, ldb), C and
 * argmax (m x n, ldc) are column-major device buffers owned by the caller;
 * work is issued on `stream` (a cudaStream_t; NULL = legacy default stream)
 * and no om_backend is needed.  Nothing is allocated: the kernel's scratch
 * lives in fixed device arrays of the library (32 MiB + 64 bytes, held on
 * every GPU that loads the library until the process exits), which limits
 * ceil(m/128) * ceil(n/64) * ceil(k/32) to 32768; larger problems on the
 * fast path fail with OM_ERR_INVALID (use om_b200_contract for them).
 * The first call on a device looks up the arrays' device addresses; make
 * that first call before any stream capture.  All calls share the arrays,
 * so calls that overlap on the GPU (other streams, other threads) race:
 * serialise them. */
int om_b200_tropical_matmul_argmax_noalloc(void* stream, om_algebra alg, int64_t m, int64_t n,
                                           int64_t k, const float* a, int64_t lda, const float* b,
                                           int64_t ldb, float* c, int64_t ldc, uint32_t* argmax);

/* ---- sequence-model operators ---------------------------------------------
 * Contractions with a step that the pairwise engine has no form for (no
 * counterpart in the reference).  Like every other call they are ordered on
 * the backend's stream, take device pointers and strides in elements, and may
 * be recorded; scratch memory comes from the backend.  They leave the
 * caller's current device as it was.  Outputs must not overlap inputs unless
 * said otherwise.  Input strides may be zero (broadcast) or negative. */

/* Gated linear recurrence along time, a chain of contractions per channel:
 *     h_t = a_t h_{t-1} + b_t,   t = 1 .. T
 *   OM_GATE_LINEAR:   a = gate,           b = x
 *   OM_GATE_SIGMOID:  a = sigmoid(gate),  b = (1 - a) x
 * gate, x and h are [D, T, B] (channels, time, batch) with shape[3] and their
 * own strides; dtype is OM_F32, OM_F64, OM_BF16 or OM_F16.  The state is kept
 * in f32 (f64 for OM_F64): h0 and h_last are contiguous [D, B] in that type;
 * h0 == NULL starts from zero, h_last (may be NULL, may be h0 itself) gets the
 * state after the last step, and h the state after every step, rounded once.
 * lengths (device, B int32, may be NULL): sequence b has
 * min(max(lengths[b], 0), T) steps; what lies behind them is not read, h is
 * zero there, and h_last is the state after the last real step.  T == 1 is the
 * form for decoding one token.
 * Steps are grouped, but the result is the definition's, also where a product of
 * gates over a group leaves the state's type or a state is infinite: such a channel
 * takes its steps one by one, which is slower.  A group's product of gates below
 * the type's smallest number counts as zero. */
typedef enum { OM_GATE_LINEAR = 0, OM_GATE_SIGMOID = 1 } om_gate;
int om_b200_gated_scan(om_backend* be, om_gate kind, om_dtype dtype, const int64_t* shape,
                       const void* gate, const int64_t* strides_gate, const void* x,
                       const int64_t* strides_x, const void* h0, const int32_t* lengths, void* h,
                       const int64_t* strides_h, void* h_last);

/* Its backward pass.  h is the forward's output, dh the gradient reaching it
 * and dh_last (contiguous [D, B] in the state's type, may be NULL) the one
 * reaching h_last.  With G_t = dh_t + a_{t+1} G_{t+1}:
 *   OM_GATE_LINEAR:   dx = G,          dgate = G h_{t-1}          (x may be NULL)
 *   OM_GATE_SIGMOID:  dx = (1 - a) G,  dgate = G (h_{t-1} - x) a (1 - a)
 * and dh0 = a_1 G_1 (contiguous [D, B], may be NULL).  dgate and dx are zero
 * behind the last step of a sequence. */
int om_b200_gated_scan_backward(om_backend* be, om_gate kind, om_dtype dtype, const int64_t* shape,
                                const void* gate, const int64_t* strides_gate, const void* x,
                                const int64_t* strides_x, const void* h, const int64_t* strides_h,
                                const void* h0, const int32_t* lengths, const void* dh,
                                const int64_t* strides_dh, const void* dh_last, void* dgate,
                                const int64_t* strides_dgate, void* dx, const int64_t* strides_dx,
                                void* dh0);

/* Softmax cross entropy of the logits z = x w^T over a vocabulary, in pieces
 * of the vocabulary and without keeping the logits:
 *     lse_n  = log sum_v exp(z_nv),   loss_n = lse_n - z_{n, targets[n]}
 * shape[3] is {D, N, V} (width, tokens, vocabulary); x is [D, N] and w [D, V]
 * with their own strides, dtype OM_F32, OM_F64, OM_BF16 or OM_F16.  targets
 * (N contiguous OM_I32 or OM_I64 values, target_dtype) outside [0, V) carry no
 * loss: loss is 0 there (lse is still written).  loss and lse are N contiguous
 * f32 values (f64 for OM_F64).  Logits may be infinite: one of -inf adds nothing
 * to lse, so a vocabulary can be masked.  16-bit products accumulate in f32.
 * f32 is computed as f32 FMA in OM_F32_EXACT mode and for one token of a width up
 * to 49144, two to four up to 12280 and five to eight up to 6136; else on the tensor
 * cores as three bf16 parts of each number: six products, error about 2^-22 *
 * sum_d |x||w|.  There a factor below 2^-109 is held to 2^-134 only, one below
 * 2^-126 may count as zero, and an infinity times an infinity is NaN. */
int om_b200_linear_cross_entropy(om_backend* be, om_dtype dtype, const int64_t* shape,
                                 const void* x, const int64_t* strides_x, const void* w,
                                 const int64_t* strides_w, om_dtype target_dtype,
                                 const void* targets, void* loss, void* lse);

/* Its gradients, from lse and the gradient dloss of each token's loss (both N
 * contiguous values): with p = exp(z - lse),
 *     dz_nv = dloss_n (p_nv - [v == targets[n]]),  dx = dz w,  dw = dz^T x
 * Tokens without a loss get dx = 0 and reach dw with nothing, whatever their row
 * of x and w hold (for the others 0 * w of an infinite w is NaN).  In the 16-bit
 * types dz is rounded to dtype before the two products, whose sums are f32. */
int om_b200_linear_cross_entropy_backward(om_backend* be, om_dtype dtype, const int64_t* shape,
                                          const void* x, const int64_t* strides_x, const void* w,
                                          const int64_t* strides_w, om_dtype target_dtype,
                                          const void* targets, const void* lse, const void* dloss,
                                          void* dx, const int64_t* strides_dx, void* dw,
                                          const int64_t* strides_dw);

/* 8-bit rows: scale_m = max_k |x_km| / 127 (f32) and
 * q_km = x_km / scale_m rounded to the nearest whole number (ties to even;
 * zero in a row of zeros).  shape[2] is {K, M}; x is [K, M] in OM_F32, OM_BF16
 * or OM_F16, q [K, M] in OM_I8, each with its own strides; scale holds M
 * values.  A row holding a NaN or an infinity gets that as its scale and only
 * zeros as q. */
int om_b200_quantize_rows(om_backend* be, om_dtype dtype, const int64_t* shape, const void* x,
                          const int64_t* strides_x, void* q, const int64_t* strides_q,
                          float* scale);

/* Matrix product in 8-bit integers with a scale for each row of q (token) and
 * of w (channel):
 *     y_nm = (sum_k q_km w_kn) q_scale_m w_scale_n + bias_n
 * shape[3] is {K, M, N}; q [K, M] and w [K, N] are OM_I8 with their own
 * strides, q_scale, w_scale and bias (may be NULL) contiguous f32, y [N, M] in
 * dtype OM_F32, OM_BF16 or OM_F16.  The sum is a 32-bit integer (K at most
 * 131071), the rest f32, rounded once. */
int om_b200_matmul_i8(om_backend* be, om_dtype dtype, const int64_t* shape, const void* q,
                      const int64_t* strides_q, const float* q_scale, const void* w,
                      const int64_t* strides_w, const float* w_scale, const float* bias, void* y,
                      const int64_t* strides_y);

/* om_b200_quantize_rows and om_b200_matmul_i8 in one call: x [K, M] and
 * y [N, M] are both of dtype. */
int om_b200_linear_i8(om_backend* be, om_dtype dtype, const int64_t* shape, const void* x,
                      const int64_t* strides_x, const void* w, const int64_t* strides_w,
                      const float* w_scale, const float* bias, void* y, const int64_t* strides_y);

#ifdef __cplusplus
}
#endif
#endif /* OMEINSUM_B200_H */
