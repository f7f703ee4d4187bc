/*
 * gear_hip.h — C ABI of libgearhip.so: the MI355X (gfx950) replay-sampling hot path of GEAR.
 *
 * Everything here is plain C: raw pointers, 64-bit sizes, a `void* stream` that is a
 * hipStream_t (NULL = the default stream).  Unless a comment says otherwise a function
 *   - returns 0 on success, a positive hipError_t on a HIP failure, or a negative
 *     GEAR_HIP_E* code on an argument error (never throws, never exits),
 *   - only enqueues work on `stream` (no device or stream synchronisation),
 *   - allocates nothing: outputs and workspaces are owned by the caller,
 *   - takes DEVICE-ACCESSIBLE pointers (hipMalloc memory, or pinned+mapped host memory for the
 *     zero-copy table case) for every array argument.
 *
 * Each entry point cites the reference interface (bigrl-team/gear, path:line) that it replaces.
 */
#ifndef GEAR_HIP_H_
#define GEAR_HIP_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define GEAR_HIP_ABI_VERSION 1

/* every entry point below is exported from libgearhip.so */
#if defined(__GNUC__)
#pragma GCC visibility push(default)
#endif

/* negative error codes (argument / usage errors detected on the host) */
#define GEAR_HIP_EINVAL (-1)      /* null pointer, negative size, inconsistent arguments     */
#define GEAR_HIP_EWORKSPACE (-2)  /* workspace pointer null or smaller than the *_bytes query */
#define GEAR_HIP_ERANGE (-3)      /* a size exceeds what the kernels index (see each call)    */
#define GEAR_HIP_EALIGN (-4)      /* a pointer that must be naturally aligned is not          */
#define GEAR_HIP_ENOTREADY (-5)   /* one-time set-up is missing and cannot run now (see call)  */

/* ---- runtime ------------------------------------------------------------------------------ */

/* ABI version of the loaded library (== GEAR_HIP_ABI_VERSION it was built with). */
int gear_hip_abi_version(void);

/* Select the HIP device for the calling thread.
 * Replaces gear::cuda::init / libgear.core.init (src/cuda/init.cu:6-18). */
int gear_hip_set_device(int device_id);

/* Number of visible HIP devices, or a negative/positive error as above in *count's place.
 * Replaces the visible_device_count probe of src/env.cc:48-53. */
int gear_hip_device_count(int *count);

/* Human-readable text for a code returned by any function of this header (static storage). */
const char *gear_hip_error_string(int code);

/* Table memory.  Replace gear::memory::CudaUVMemory::alloc/free (src/memory/cuda_uvm.cc:10-54:
 * cudaHostAlloc mapped|portable) and gear::memory::CudaMemory (src/memory/cuda_memory.cc:6-28).
 * These four DO allocate / free and may synchronise; they are set-up calls, not hot-path calls.
 * gear_hip_host_alloc returns pinned host memory that the GPU reads in place (zero-copy);
 * *dev_ptr receives the device-side alias of the same bytes. */
int gear_hip_host_alloc(size_t bytes, void **host_ptr, void **dev_ptr);
int gear_hip_host_free(void *host_ptr);
int gear_hip_device_alloc(size_t bytes, void **dev_ptr);
int gear_hip_device_free(void *dev_ptr);

/* Blocking copy of `bytes` between any two of host / pinned / device memory (direction inferred
 * from the pointers).  A set-up call for filling and reading back device-resident tables
 * (stands where Span::copy uses memcpy on the host-resident table, include/common/span.h:73-79). */
int gear_hip_memcpy(void *dst, const void *src, size_t bytes);

/* Pin + map an existing host range (SysV shared memory segment of a TrajectoryTable).
 * Replaces the cudaHostRegister(Mapped|Portable) of gear::memory::SharedMemory::alloc
 * (src/memory/shared_memory.cc:59-61) and the cudaHostUnregister of ::free (:70).
 * Some ROCm installations refuse registration of existing memory; the error is returned and
 * the caller falls back to gear_hip_host_alloc. */
int gear_hip_host_register(void *host_ptr, size_t bytes, void **dev_ptr);
int gear_hip_host_unregister(void *host_ptr);

/* ---- trajectory-window gather ------------------------------------------------------------- */

/* Fused window arithmetic + byte gather of one column.
 * Replaces gear::cuda::launch_fused_subcopy_collect + fused_subcopy_collect
 * (src/cuda/copy.cu:91-134,217-242) as called by CpuTrajectoryStorageHandler::fused_subcopy
 * (src/storage/handler.cc:133-154) behind libgear.core handler.subcopy
 * (src/storage/pybind.cc:140-146).
 *
 * For window g in [0,num):
 *     lsub = max(tss[g] + ofst, 0);  rsub = min(lsub + span, lens[g]);
 *     n    = max(rsub - lsub, 0) * step_bytes;
 *     npad = pad_head ? dst_stride - n : 0;
 *     dst[g*dst_stride + npad .. +n) = src[idxs[g]*traj_stride + col_base + lsub*step_bytes .. +n)
 * src       table base (HBM, or pinned mapped host memory: the zero-copy path)
 * dst       contiguous [num, dst_stride] bytes, 16-byte aligned (any torch tensor is)
 * idxs/tss/lens  int64[num] on the device: trajectory index, timestep, trajectory length
 * traj_stride    bytes per trajectory (T * sum of per-step column bytes; src/storage/table.cc:14-16)
 * step_bytes     bytes per step of this column (ColumnSpec::size, src/storage/specs.cc:10-14)
 * col_base       accu_stride(column) * T (src/storage/handler.cc:143-145)
 * dst_stride     bytes per window in dst (pattern.length * step_bytes, handler.cc:146-147)
 * zero_fill      0: padding bytes of dst are left untouched, as in the reference (whose caller
 *                pre-zeroes the batch with torch.zeros, gear/loader/offline_loader.py:181-189);
 *                1: the kernel writes the padding zeros itself, so dst may be uninitialised.
 * mask_out       NULL, or uint8[num, span] on the device: 1 where the step holds copied data,
 *                0 where it is padding (no reference counterpart; benchmark config 3's mask).
 * All offsets are 64-bit (the reference's kernel truncates them to int, copy.cu:93-115).
 * Requires n <= dst_stride for every window (GEAR_HIP_EINVAL if span*step_bytes > dst_stride). */
int gear_hip_subcopy(const void *src, void *dst, int64_t num, const int64_t *idxs,
                     const int64_t *tss, const int64_t *lens, int pad_head, int64_t ofst,
                     int64_t span, int64_t traj_stride, int64_t step_bytes, int64_t col_base,
                     int64_t dst_stride, int zero_fill, uint8_t *mask_out, void *stream);

/* One launch for several columns of the same batch of windows (no reference counterpart as an
 * entry point: it is the per-column loop of OfflineLoader.fused_iterate,
 * gear/loader/offline_loader.py:178-203, folded into one grid).
 * cols points to `ncols` descriptors in HOST memory (copied into kernel arguments). */
typedef struct gear_hip_column_desc {
  void *dst;          /* [num, dst_stride] bytes on the device, 16-byte aligned */
  uint8_t *mask_out;  /* NULL or uint8[num, span] */
  int64_t ofst, span; /* SubscribePattern offset / length (include/storage/handler.h:17-31) */
  int64_t step_bytes, col_base, dst_stride;
  int32_t pad_head, zero_fill;
} gear_hip_column_desc;
#define GEAR_HIP_MAX_COLUMNS 16
int gear_hip_subcopy_multi(const void *src, int64_t num, const int64_t *idxs, const int64_t *tss,
                           const int64_t *lens, int64_t traj_stride,
                           const gear_hip_column_desc *cols, int ncols, void *stream);

/* The same launch with the batch checked against the table on the device: a window whose
 * trajectory index lies outside [0, capacity) reads nothing (its rows are all padding, its mask
 * all 0) and lens[g] is clamped to trajectory_length, so no index a caller passes can make the
 * kernel read outside the table.  The reference's kernel trusts its inputs
 * (src/cuda/copy.cu:110-123); capacity = 0 / trajectory_length = 0 switch the respective check
 * off, which is what gear_hip_subcopy_multi does. */
int gear_hip_subcopy_multi_checked(const void *src, int64_t num, const int64_t *idxs,
                                   const int64_t *tss, const int64_t *lens, int64_t traj_stride,
                                   int64_t capacity, int64_t trajectory_length,
                                   const gear_hip_column_desc *cols, int ncols, void *stream);

/* Generic slice gather: dst[dst_offsets[g] .. +strides[g]) = src[src_offsets[g] .. +strides[g]).
 * Replaces launch_vary_stride_copy_collect / vary_stride_copy_collect
 * (src/cuda/copy.cu:47-89,175-215; libgear.core.vcopy / copy_debug, copy.cu:247-258).
 * strides[g] <= max_stride must hold; slices with strides[g] <= 0 copy nothing.
 * Any byte alignment of src/dst offsets is accepted (the reference requires 16 B). */
int gear_hip_vcopy(const void *src, void *dst, int64_t num, const int64_t *src_offsets,
                   const int64_t *dst_offsets, const int64_t *strides, int64_t max_stride,
                   void *stream);

/* Same with one fixed slice length.  Replaces launch_fix_stride_copy_collect /
 * fix_stride_copy_collect (src/cuda/copy.cu:12-45,138-173; libgear.core.copy, copy.cu:246). */
int gear_hip_copy(const void *src, void *dst, int64_t num, const int64_t *src_offsets,
                  const int64_t *dst_offsets, int64_t stride, void *stream);

/* Device-side restatement of CpuTrajectoryStorageHandler::sub (src/storage/handler.cc:78-131):
 * fills src_offsets/dst_offsets/copy_lens (int64[num], device) from idxs/tss/lens without the
 * host loop and the three H2D copies of gear/loader/offline_loader.py:260-277. */
int gear_hip_sub(int64_t num, const int64_t *idxs, const int64_t *tss, const int64_t *lens,
                 int pad_head, int64_t ofst, int64_t span, int64_t traj_stride,
                 int64_t step_bytes, int64_t col_base, int64_t *src_offsets,
                 int64_t *dst_offsets, int64_t *copy_lens, void *stream);

/* Sampled flat step index -> window arguments of gear_hip_subcopy, for tables whose priorities
 * are kept per step (benchmark configs 4 and 5):  f = flat[j] (mod `modulo` when modulo > 0);
 *     idxs[j] = f / trajectory_length;  tss[j] = f % trajectory_length;  lens[j] = tss[j] + 1
 * (lens may be NULL).  lens = ts + 1 is the offline convention "timestep == length" of
 * gear/loader/offline_loader.py:200-201,263 applied to a step inside a trajectory: the window
 * never reaches past the sampled step.  Stands where the loader looks timesteps up on the host
 * (gear/loader/offline_loader.py:168-177). */
int gear_hip_split_step_index(const int64_t *flat, int64_t num, int64_t trajectory_length,
                              int64_t modulo, int64_t *idxs, int64_t *tss, int64_t *lens,
                              void *stream);

/* out[j] = table[idx[j]] + add for int64 tables on the device (0 where idx[j] is outside [0,n)).
 * Replaces the host-side look-ups of the sampled batch: iset.timesteps[indices.cpu()]
 * (gear/loader/offline_loader.py:168-177) and concat_indices[draws]
 * (gear/sampler/global_sampler.py:131,172,196). */
int gear_hip_take_i64(const int64_t *table, int64_t n, const int64_t *idx, int64_t num,
                      int64_t add, int64_t *out, void *stream);

/* ---- weighted sampler: prefix sum + search ------------------------------------------------ */

/* Inclusive prefix sum of fp32 priorities accumulated and written in fp64:
 *     out[i] = sum_{j<=i} (double) in[j]
 * One pass over the input for up to 16384 ranges (n <= 268 M fp32, 134 M int64): every workgroup publishes
 * the sum of its range and adds the sums of all earlier ranges -- beyond 6656 ranges those of the earlier ones of its
 * group of 64 and of all earlier groups --, with a bounded wait (a workgroup that waited too long sums the missing
 * range itself and publishes it: same bits, no kernel can hang).  For a stream under graph capture and with
 * GEAR_HIP_SCAN_SINGLE_PASS=0: two launches (range sums, then the scan) up to 6656 ranges, three (the groups' sums
 * in between) up to 16384.  More ranges: three launches (the ranges' prefix in between).  fp32 beyond 33.5 M is cut
 * into ranges of 16384 elements, int64 beyond 16.8 M into 8192, or 4096 where it takes several launches.  The result
 * is bit-identical in all cases and on every run.  Replaces
 * gear::cuda::launch_prefix_sum /
 * one_dimension_prefix_sum (src/cuda/one_dim_prefix_sum.cu:125-273; libgear.core.prefix_sum,
 * :276-278), which is fp32 and only correct for one block.
 * workspace: device memory of at least gear_hip_scan_workspace_bytes(n) bytes, 256-byte aligned;
 * its contents need not be initialised (the call initialises it on `stream`).
 * n may be 0 (nothing is written).  n <= 2^40.  `out` must be 16-byte aligned.
 * One workspace serves one call at a time.  Two one-pass calls that share a workspace while both
 * run cannot hang (the wait is bounded) but may find each other's words; a range that could not
 * be completed is marked: its prefixes are NaN (fp64 / fp32 results) or start from INT64_MIN
 * (gear_hip_scan_i64: negative results where the inputs are not).
 * Rounding: inside a range (2048, 4096 or 8192 elements, by n) the prefix is a running sum of a
 * fixed association; the offset of a range is the separately rounded sum of all earlier ranges.
 * Both are within 1e-12 (relative) of the sequential fp64 sum, but they are rounded differently,
 * so across a range boundary out[i+1] can fall below out[i] + in[i+1] by an ulp or two of the
 * running total; with non-negative input the result is still non-decreasing except where that
 * difference exceeds in[i+1] (inputs below ~1e-16 of the total). */
size_t gear_hip_scan_workspace_bytes(int64_t n);
int gear_hip_scan_f32_f64(const float *in, double *out, int64_t n, void *workspace,
                          size_t workspace_bytes, void *stream);

/* gear_hip_scan_f32_f64 for callers that cannot allocate device memory: code under HIP graph
 * capture, tight serving loops, harnesses with a frozen memory pool.  It has no counterpart in
 * the reference.  The range sums that the other entry point keeps in the caller's workspace live
 * in a static device array inside the library (about 2 MiB per GPU, held until the process ends);
 * the call allocates and frees nothing.  Same result, bit for bit, as gear_hip_scan_f32_f64.
 * n <= gear_hip_scan_static_max_n() (2^27 = 134 217 728), else GEAR_HIP_ERANGE.
 * The array's address is looked up once per device, by gear_hip_set_device or by the first call
 * on that device; a first call on a stream that is being captured cannot look it up and returns
 * GEAR_HIP_ENOTREADY (call gear_hip_set_device, or once outside the capture, first).
 * All calls on one GPU share the array.  Outside graph capture the library orders them itself:
 * a call's kernels wait (on the device, through an event) for the kernels of the previous static
 * call on that GPU, whatever stream or host thread that one came from.  Captured calls are not
 * ordered by the library: graphs that hold one must not run at the same time as another static
 * call on that GPU, or the two race on the array; use the workspace form there. */
int64_t gear_hip_scan_static_max_n(void);
int gear_hip_scan_f32_f64_static(const float *in, double *out, int64_t n, void *stream);

/* Incremental form for the online priority path (priorities of a few trajectories change between
 * batches: SharedMemoryIndexServer::update, src/index/server.cc:175-180, and
 * WeightUpdateRequestArray, src/index/request.cc:41-75; the reference has no prefix to maintain).
 * Preconditions: the last call on (in, out, workspace) was gear_hip_scan_f32_f64 or this function
 * with the same n, and since then only in[first_changed .. n) changed.  Then out[i] is
 * recomputed from the start of the range that holds first_changed onwards, reusing the range sums
 * kept in the workspace; the result is bit-identical to a full gear_hip_scan_f32_f64.
 * first_changed >= n: nothing to do; first_changed = 0: a full scan. */
int gear_hip_rescan_f32_f64(const float *in, double *out, int64_t n, int64_t first_changed,
                            void *workspace, size_t workspace_bytes, void *stream);

/* The same scan (fp64 accumulation) with the result rounded to fp32 on output: the signature of
 * the reference's binding, prefix_sum(FloatTensor input, FloatTensor output)
 * (src/cuda/one_dim_prefix_sum.cu:246-278). */
int gear_hip_scan_f32_f32(const float *in, float *out, int64_t n, void *workspace,
                          size_t workspace_bytes, void *stream);

/* Same scan over int64 weights (trajectory lengths, include/index/set.h:42), exact in int64
 * (two's complement: weights of either sign, sums wrap like int64 additions).
 * Used for length-weighted trajectory sampling (benchmark config 3).
 * n <= 2^40. */
int gear_hip_scan_i64(const int64_t *in, int64_t *out, int64_t n, void *workspace,
                      size_t workspace_bytes, void *stream);

/* Sum of n fp32 values accumulated in fp64, written to out[0] (device) as fp32 and, when
 * out_f64 is not NULL, as fp64 to out_f64[0].  Deterministic (fixed reduction tree).
 * Replaces gear::cuda::launch_sum / one_dimension_sum (src/cuda/one_dim_sum.cu:22-99;
 * libgear.core.sum, :102-104), which uses fp32 atomics on the default stream.
 * workspace: gear_hip_sum_workspace_bytes(n) bytes on the device. */
size_t gear_hip_sum_workspace_bytes(int64_t n);
int gear_hip_sum_f32(const float *in, int64_t n, float *out, double *out_f64, void *workspace,
                     size_t workspace_bytes, void *stream);

/* Batched upper_bound of draws in an fp64 inclusive prefix array:
 *     idx_out[j] = min( #{ i : prefix[i] <= t_j }, n-1 )
 * with t_j = (double) u[j]                       when unit_uniforms == 0 (u in [0, total)),
 *      t_j = (double) u[j] * prefix[n-1]         when unit_uniforms != 0 (u in [0, 1)).
 * This is the "binary search of seeded uniforms" half of the weighted sampler (no kernel in
 * the reference; it stands where WeightedSampler calls torch.multinomial,
 * gear/sampler/global_sampler.py:170).
 * Optional importance weights (both or neither of priorities / weights_out non-NULL):
 *     w_j = ( n * priorities[idx_j] / prefix[n-1] ) ^ (-beta), computed in fp64;
 *     weights_out[j] = (float)( w_j / max_j w_j ).
 * workspace: gear_hip_search_workspace_bytes(num) bytes on the device (only used for weights;
 * may be NULL/0 when weights_out is NULL). */
size_t gear_hip_search_workspace_bytes(int64_t num);
int gear_hip_upper_bound_f64(const double *prefix, int64_t n, const float *u, int64_t num,
                             int unit_uniforms, int64_t *idx_out, const float *priorities,
                             double beta, float *weights_out, void *workspace,
                             size_t workspace_bytes, void *stream);

/* The sampler of one batch in one call: draws searched in the fp64 prefix (as
 * gear_hip_upper_bound_f64), the found indices sorted ascending -- what every sampler of the
 * reference returns, torch.sort(...).values, gear/sampler/global_sampler.py:131,172,195-199 --
 * and, when trajectory_length > 0, split like gear_hip_split_step_index into idxs/tss/lens
 * (lens may be NULL).  sorted_out may be NULL when trajectory_length > 0.
 * Up to 32768 draws take one launch (search, order and split); larger batches, and outputs that lie on
 * top of the draws or the prefix, a search, a sort and a split of their own.
 * workspace: gear_hip_sample_workspace_bytes(num) bytes on the device. */
size_t gear_hip_sample_workspace_bytes(int64_t num);
int gear_hip_sample_sorted_f64(const double *prefix, int64_t n, const float *u, int64_t num,
                               int unit_uniforms, int64_t *sorted_out, int64_t trajectory_length,
                               int64_t modulo, int64_t *idxs, int64_t *tss, int64_t *lens,
                               void *workspace, size_t workspace_bytes, void *stream);

/* Batch selection with the look-ups the loader performs before it can gather, in one call.
 * For a batch of positions into the loader's index array, sorted ascending, the entry at sorted
 * place r with position p yields
 *     sampled_out[r] = index_table ? index_table[p] : p      (0 for p outside [0, index_n))
 *     local_out[r]   = sampled_out[r] - index_offset
 *     lens_out[r]    = lengths_table[local_out[r]]            (0 outside [0, lengths_n))
 * Any of the three outputs may be NULL (not all); lens_out needs lengths_table.  This replaces,
 * for a sampler whose index array ascends (then sort(indices[p]) == indices[sort(p)]), the chain
 * torch.sort(concat_indices[draws]) (gear/sampler/global_sampler.py:131,172,196),
 * indices - index_offset and iset.timesteps[indices.cpu()] on the host
 * (gear/loader/offline_loader.py:161-177): up to 32768 positions or draws take ONE launch (search,
 * order and look-ups), more take the radix sort and an element-wise launch; so do many among a few
 * entries, and outputs that lie on top of the draws, the prefix or the positions.
 *   gear_hip_sample_lookup_f64  positions = upper_bound of the draws u in the fp64 prefix, as
 *                               gear_hip_upper_bound_f64 (index_table, when given, has n entries)
 *   gear_hip_sample_lookup_i64  the same in an int64 prefix (a sampler over lengths), u as for
 *                               gear_hip_upper_bound_i64; with starts_out, also the start of a
 *                               window of `window` steps inside the entry's recorded length:
 *                               starts_out[r] = floor(start_uniforms[r] * (lens[r] - window + 1)),
 *                               0 where the length is below the window (start_uniforms: num
 *                               doubles in [0, 1); needs lengths_table; starts_out may be NULL)
 *   gear_hip_sort_lookup_i64    positions given (uniform draws), each in [0, bound)
 *   gear_hip_lookup_i64         positions given and already in the wanted order (the top-k's
 *                               index-ordered selection): look-ups only, no workspace
 * workspace: gear_hip_sample_workspace_bytes(num) bytes on the device. */
int gear_hip_sample_lookup_f64(const double *prefix, int64_t n, const float *u, int64_t num,
                               int unit_uniforms, const int64_t *index_table,
                               int64_t index_offset, const int64_t *lengths_table,
                               int64_t lengths_n, int64_t *sampled_out, int64_t *local_out,
                               int64_t *lens_out, void *workspace, size_t workspace_bytes,
                               void *stream);
int gear_hip_sample_lookup_i64(const int64_t *prefix, int64_t n, const void *u, int64_t num,
                               int unit_uniforms, const int64_t *index_table,
                               int64_t index_offset, const int64_t *lengths_table,
                               int64_t lengths_n, int64_t *sampled_out, int64_t *local_out,
                               int64_t *lens_out, const double *start_uniforms, int64_t window,
                               int64_t *starts_out, void *workspace, size_t workspace_bytes,
                               void *stream);
int gear_hip_sort_lookup_i64(const int64_t *positions, int64_t num, int64_t bound,
                             const int64_t *index_table, int64_t index_n, int64_t index_offset,
                             const int64_t *lengths_table, int64_t lengths_n,
                             int64_t *sampled_out, int64_t *local_out, int64_t *lens_out,
                             void *workspace, size_t workspace_bytes, void *stream);
int gear_hip_lookup_i64(const int64_t *positions, int64_t num, const int64_t *index_table,
                        int64_t index_n, int64_t index_offset, const int64_t *lengths_table,
                        int64_t lengths_n, int64_t *sampled_out, int64_t *local_out,
                        int64_t *lens_out, void *stream);

/* Same search in an int64 prefix array (exact): t_j = floor(u[j] * prefix[n-1]) with u fp64 in
 * [0,1) when unit_uniforms != 0, else t_j = (int64) u[j] taken from an int64 array passed
 * through `u` (cast).  idx_out[j] = min(#{i : prefix[i] <= t_j}, n-1). */
int gear_hip_upper_bound_i64(const int64_t *prefix, int64_t n, const void *u, int64_t num,
                             int unit_uniforms, int64_t *idx_out, void *stream);

/* ---- sort / top-k / priority update ------------------------------------------------------- */

/* gear_hip_sample_lookup_f64 for uniforms, and gear_hip_sort_lookup_i64 for integers in [0, bound), that the
 * call draws itself: the numbers that torch's GPU generator of this seed and offset gives to one rand
 * (float32) or randint (int64) call of `num` elements (Philox4x32-10; the caller advances the offset by 4).
 * num <= gear_hip_draw_max() -- as many as the current GPU holds threads at once, gear_hip_draw_max_of(its compute
 * units, threads apiece): torch numbers the elements of larger calls in another way --,
 * bound <= gear_hip_draw_max_bound() (2^28 - 1: from 2^28 on torch's randint takes two words a draw), else
 * GEAR_HIP_ERANGE.  They take the place of the torch.randint and torch.multinomial of
 * gear/sampler/global_sampler.py:121-199. */
int64_t gear_hip_draw_max(void);
int64_t gear_hip_draw_max_of(int compute_units, int threads_per_unit);
int64_t gear_hip_draw_max_bound(void);
int gear_hip_draw_lookup_f64(const double *prefix, int64_t n, uint64_t seed, uint64_t offset, int64_t num,
                             const int64_t *index_table, int64_t index_offset,
                             const int64_t *lengths_table, int64_t lengths_n, int64_t *sampled_out,
                             int64_t *local_out, int64_t *lens_out, void *workspace,
                             size_t workspace_bytes, void *stream);
int gear_hip_draw_sort_lookup_i64(uint64_t seed, uint64_t offset, int64_t num, int64_t bound,
                                  const int64_t *index_table, int64_t index_n, int64_t index_offset,
                                  const int64_t *lengths_table, int64_t lengths_n, int64_t *sampled_out,
                                  int64_t *local_out, int64_t *lens_out, void *workspace,
                                  size_t workspace_bytes, void *stream);

/* Ascending sort (by counting, or LSD radix) of `num` int64 keys (non-negative, < 2^key_bits) with an optional
 * int64 payload, stable.  keys_out/vals_out must not alias the inputs.
 * Replaces the torch.sort of sampled indices in every sampler
 * (gear/sampler/global_sampler.py:131,172,195-199) and the unfinished
 * include/cuda/sort.cuh:19-122.
 * workspace: gear_hip_sort_workspace_bytes(num) bytes on the device. */
size_t gear_hip_sort_workspace_bytes(int64_t num);
int gear_hip_sort_i64(const int64_t *keys_in, int64_t *keys_out, const int64_t *vals_in,
                      int64_t *vals_out, int64_t num, int key_bits, void *workspace,
                      size_t workspace_bytes, void *stream);

/* The entries table[idx[j]] (0 for an index outside [0, n)) in ascending order of their low 63 bits, stable: what
 * gear_hip_take_i64 and gear_hip_sort_i64 give.  For entries that are in order already more often than not
 * (ascending positions in a table that is usually ascending too): up to 32768 of them, the sort is a launch
 * that finds nothing to do.  out must not alias the inputs.
 * workspace: gear_hip_take_sorted_workspace_bytes(num) bytes on the device. */
size_t gear_hip_take_sorted_workspace_bytes(int64_t num);
int gear_hip_take_sorted_i64(const int64_t *table, int64_t n, const int64_t *idx, int64_t num, int64_t *out,
                             void *workspace, size_t workspace_bytes, void *stream);

/* Top-k of fp32 priorities, largest first; among equal priorities the smaller index wins
 * (i.e. the first k entries of a stable descending sort).  NaN is not a valid priority.
 * Replaces torch.topk(weights, k, largest=True) of TopKSampler
 * (gear/sampler/global_sampler.py:195-199) and the dead include/cuda/sort.cuh.
 *   sorted_by_value != 0: values_out/indices_out ordered by (value desc, index asc)
 *   sorted_by_value == 0: the same set ordered by index ascending (what TopKSampler returns
 *                         after its torch.sort of the indices)
 * values_out may be NULL.  1 <= k <= n < 2^31.
 * The priorities are normally read once: a sample of 2048 of them places a bound safely below
 * the k-th largest, the one pass over the array lists everything above the bound, and the exact
 * selection runs on those lists.  Where a list overflows (clustered maxima, masses of ties) the
 * later steps read that part of the array again; where the bound fails (fewer than k entries
 * above it: a sample that misleads) two of them read all of it again and look for the threshold
 * among the entries below the bound.  The result is the same either way.
 * workspace: gear_hip_topk_workspace_bytes(n, k) bytes on the device, 256-byte aligned; its
 * contents need not be initialised (the call clears what it needs on `stream`). */
size_t gear_hip_topk_workspace_bytes(int64_t n, int64_t k);
int gear_hip_topk_f32(const float *priorities, int64_t n, int64_t k, int sorted_by_value,
                      float *values_out, int64_t *indices_out, void *workspace,
                      size_t workspace_bytes, void *stream);

/* The same selection for a caller that repeats it on a slowly changing array (the priority
 * maintenance of a replay buffer between batches: TopKSampler.sync_sample on every step,
 * gear/sampler/global_sampler.py:175-203, after the updates of src/index/request.cc:41-51).
 * Every call leaves in the workspace the bound the NEXT call can start from: the boundary at or
 * below the 2k-th largest priority, taken from this call's exact counts.  This form takes that
 * bound up instead of drawing a sample when `workspace` was last used by gear_hip_topk_f32 or
 * this function with the same n, k and order (a mark in the workspace says so; anything else in
 * it, and a call whose own bound failed, lead to a sample as in gear_hip_topk_f32).  The bound
 * only decides how the work is done: however stale it is, the result equals gear_hip_topk_f32's
 * bit for bit (too high: the entries below it are searched as described above; too low: lists
 * overflow and those parts of the array are read again). */
int gear_hip_topk_f32_warm(const float *priorities, int64_t n, int64_t k, int sorted_by_value,
                           float *values_out, int64_t *indices_out, void *workspace,
                           size_t workspace_bytes, void *stream);

/* Priority update  weights[idx[j]] = values[j], j in [0,num).
 * Replaces the host loop over Indexset::set_weight (include/index/set.h:245-247) and fixes the
 * semantics of WeightUpdateRequestArray::update (src/index/request.cc:41-51): when an index
 * occurs more than once the LAST occurrence wins.
 *   unique_indices != 0: caller guarantees no duplicates; plain scatter, no workspace needed.
 *   unique_indices == 0: duplicates resolved deterministically (a hash table of the indices, or a
 *                        stable radix sort of them); workspace of gear_hip_scatter_workspace_bytes(num) bytes.
 * Indices outside [0,n) are ignored. */
size_t gear_hip_scatter_workspace_bytes(int64_t num);
int gear_hip_scatter_f32(float *weights, int64_t n, const int64_t *idx, const float *values,
                         int64_t num, int unique_indices, void *workspace,
                         size_t workspace_bytes, void *stream);

/* The same update for int64 tables: timesteps[idx[j]] = values[j] (the trajectory lengths that
 * travel with the priorities in a weight-update request, src/index/server.cc:175-180,
 * Indexset::set_timestep, include/index/set.h:242-244).  Same workspace query. */
int gear_hip_scatter_i64(int64_t *table, int64_t n, const int64_t *idx, const int64_t *values,
                         int64_t num, int unique_indices, void *workspace, size_t workspace_bytes,
                         void *stream);

/* ---- a batch of windows into a sequence model ---------------------------------------------- */

/* The calls of this part have no counterpart in the reference: they are what a sequence model of
 * trajectories does with the batches of gear/loader/offline_loader.py:155-204. */

/* element types of the calls below */
#define GEAR_HIP_F32 0
#define GEAR_HIP_F16 1
#define GEAR_HIP_BF16 2

/* Ranges of keys and positions of a batch of windows, from the loader's validity masks and a
 * `done` column.  Step s of window b is valid where mask[b][s] != 0 (mask NULL: all are).  A
 * document is a maximal run of valid steps without a done (done NULL: none) before its last step;
 * it covers the steps [s0, s1).  A step is `tokens_per_step` tokens n; token i = s*n + u sees the
 * keys lo[b][i] <= j < hi[b][i]:
 *     lo = s0*n
 *     hi = i+1 (GEAR_HIP_RANGE_CAUSAL), (s+1)*n (_STEP), s1*n (_DOCUMENT),
 *          and max(hi, min(s0 + prefix, s1)*n) where prefix > 0 (the first steps see each other)
 * Tokens of steps that are not valid get lo = hi = 0 and position 0.  pos is [batch][steps*n][axes]:
 * s - s0 (axes = 1), or with grid_rows, grid_cols > 0 and n = grid_rows*grid_cols the three
 * positions s - s0, u / grid_cols, u % grid_cols.  steps * n < 2^31, else GEAR_HIP_ERANGE. */
#define GEAR_HIP_RANGE_CAUSAL 0
#define GEAR_HIP_RANGE_STEP 1
#define GEAR_HIP_RANGE_DOCUMENT 2
int gear_hip_token_ranges(const uint8_t *mask, const uint8_t *done, int64_t batch, int64_t steps,
                          int64_t tokens_per_step, int mode, int64_t prefix, int64_t grid_rows,
                          int64_t grid_cols, int32_t *lo, int32_t *hi, int32_t *pos, void *stream);

/* Norm of every head's query and key with the rotation of its positions, in one pass.  For a row x
 * of head_dim D elements, y = x / sqrt(mean(x^2) + eps) * weight; the pair (y[i], y[i + D/2]) is
 * turned by the angle pos[axis(i)] * freqs[i].  The first sections[0] pairs belong to axis 0, the
 * next sections[1] to axis 1, ...; pairs beyond the sections are not turned.  All arithmetic is
 * in 32 bits, the angles are reduced to a turn in 64, so that any int32 position is exact.
 *   head_dim       a multiple of 16, at most 256
 *   q, k           batch x tokens x heads x head_dim, the innermost contiguous; strides of batch,
 *                  token and head in elements; bases and strides multiples of 16 bytes
 *   q_weight, k_weight   head_dim elements of type f32 (weight_f32 != 0) or of the rows' type,
 *                  or NULL: ones */
typedef struct gear_hip_norm_rotate_desc {
  const void *q, *k;
  int64_t q_stride[3], k_stride[3];
  int64_t batch, tokens;
  int32_t q_heads, k_heads, head_dim, dtype;
  const int32_t *pos;  /* [batch][tokens][axes] */
  const double *freqs; /* [sum of sections], radians a position */
  int32_t axes, sections[4];
  int32_t weight_f32;
  const void *q_weight, *k_weight;
  float eps;
} gear_hip_norm_rotate_desc;
/* q_out, k_out: contiguous, of the inputs' type */
int gear_hip_norm_rotate(const gear_hip_norm_rotate_desc *desc, void *q_out, void *k_out,
                         void *stream);
/* The same for the newest tokens of rollouts: the result of k and the rows of v (as k) go to row
 * slots[b][t] of the caches [batch][cache_tokens][k_heads][head_dim] (strides of batch, token and
 * head as above); a slot outside [0, cache_tokens) is not written. */
int gear_hip_norm_rotate_append(const gear_hip_norm_rotate_desc *desc, const void *v,
                                const int64_t *v_stride, void *q_out, const int32_t *slots,
                                int64_t cache_tokens, void *k_cache, const int64_t *k_cache_stride,
                                void *v_cache, const int64_t *v_cache_stride, void *stream);
/* Gradients of gear_hip_norm_rotate: dq, dk (contiguous) from dq_out, dk_out (strides as above),
 * and of the weights (of the weights' type, summed in 32 bits in a fixed order; NULL: not wanted).
 * workspace: gear_hip_norm_rotate_backward_workspace_bytes(head_dim) bytes on the device. */
size_t gear_hip_norm_rotate_backward_workspace_bytes(int64_t head_dim);
int gear_hip_norm_rotate_backward(const gear_hip_norm_rotate_desc *desc, const void *dq_out,
                                  const int64_t *dq_out_stride, const void *dk_out,
                                  const int64_t *dk_out_stride, void *dq, void *dk,
                                  void *dq_weight, void *dk_weight, void *workspace,
                                  size_t workspace_bytes, void *stream);

/* Attention in which query i sees the keys lo[b][i] <= j < hi[b][i] (as gear_hip_token_ranges
 * gives them; ranges are cut to [0, keys)):
 *     s_ij = scale * q_i . k_j;   cap > 0: s_ij = cap * tanh(s_ij / cap);
 *     slopes != NULL: s_ij -= slopes[head] * |i + keys - queries - j|
 *     p_ij = softmax of s_ij over the keys seen;  out_i = sum_j p_ij v_j;  lse_i = log sum_j exp s_ij
 * A query that sees nothing gets out = 0, lse = -inf, and passes no gradient on; what its row of q
 * (and of dout) holds is not looked at.  Head h reads key head h / (heads / kv_heads).
 * Scores, statistics and sums are held in 32 bits; p (and its gradient) is rounded to the inputs'
 * type where it is multiplied with rows of that type.
 *   dtype     GEAR_HIP_F16 or GEAR_HIP_BF16; head_dim a multiple of 16, at most 128
 *   q, k, v   batch x queries|keys x heads|kv_heads x head_dim, the innermost contiguous; strides
 *             of batch, token and head in elements; bases and strides multiples of 16 bytes
 *   queries, keys < 2^30, and less than 2^32 work items a launch, else GEAR_HIP_ERANGE: batch * heads * (queries / 128, rounded
 *   up) and batch * kv_heads * (keys / 128, rounded up) below 2^24, for steps batch * kv_heads *
 *   (queries * heads / kv_heads / 32, rounded up) below 2^24;  0 < scale < 1e30;  cap 0 (none), or below 1e30 and above 1e-30 scale */
typedef struct gear_hip_attention_desc {
  const void *q, *k, *v;
  int64_t q_stride[3], k_stride[3], v_stride[3];
  int64_t batch, queries, keys;
  int32_t heads, kv_heads, head_dim, dtype;
  const int32_t *lo, *hi; /* [batch][queries] */
  const float *slopes;    /* [heads] or NULL */
  float scale, cap;
} gear_hip_attention_desc;
/* out: [batch][queries][heads][head_dim] contiguous; lse: [batch][heads][queries] (NULL: not wanted) */
int gear_hip_attention(const gear_hip_attention_desc *desc, void *out, float *lse, void *stream);
/* Gradients dq, dk, dv (contiguous, laid out as q, k, v) from dout (strides as above) and the
 * forward call's out and lse.  No atomics: the same bits on every run.
 * workspace: gear_hip_attention_backward_workspace_bytes(batch, queries, heads) bytes, 256-byte aligned. */
size_t gear_hip_attention_backward_workspace_bytes(int64_t batch, int64_t queries, int64_t heads);
int gear_hip_attention_backward(const gear_hip_attention_desc *desc, const void *dout,
                                const int64_t *dout_stride, const void *out, const float *lse,
                                void *dq, void *dk, void *dv, void *workspace,
                                size_t workspace_bytes, void *stream);
/* The same attention for the newest tokens of rollouts over their caches (k, v: batch x keys =
 * cache rows): few queries, each with the range of its own rollout.  The distance is counted from
 * the last key that a query sees: |hi - 1 - j|.  The keys are split over workgroups and joined.
 * workspace: gear_hip_attention_step_workspace_bytes(batch, queries, keys, heads, kv_heads,
 * head_dim) bytes on the device, 256-byte aligned. */
size_t gear_hip_attention_step_workspace_bytes(int64_t batch, int64_t queries, int64_t keys,
                                               int64_t heads, int64_t kv_heads, int64_t head_dim);
int gear_hip_attention_step(const gear_hip_attention_desc *desc, void *out, void *workspace,
                            size_t workspace_bytes, void *stream);

/* ---- tokens: into a sequence model and out of it ---------------------------------------------- */

/* These have no counterpart in the reference either: they are what stands at both ends of a sequence model whose
 * observations and actions are tokens, and between its blocks.  Tokens are int64 (tokens_i64 != 0) or int32; a token
 * outside [0, vocab) stands for none (padding).  Rows are `width` or `vocab` contiguous elements of one of the types
 * above, at any stride (in elements) and any element's address; results are contiguous.  Sums and statistics are held
 * in 32 bits, results are rounded once, and no call uses atomics on results: the same bits on every run. */

/* out[i] = scale * table[tokens[i]], zeros where there is no token.  n, vocab < 2^31 - 1, width <= 2^20. */
int gear_hip_embed(const void *tokens, int tokens_i64, int64_t n, const void *table, int64_t table_stride,
                   int64_t vocab, int64_t width, int dtype, float scale, void *out, void *stream);
/* dtable[v] = scale * (sum over i with tokens[i] = v of dout[i]), all of [vocab][width] written, in the type of dout.
 * workspace: gear_hip_embed_backward_workspace_bytes(n, width) bytes on the device, 16-byte aligned. */
size_t gear_hip_embed_backward_workspace_bytes(int64_t n, int64_t width);
int gear_hip_embed_backward(const void *dout, int64_t dout_stride, const void *tokens, int tokens_i64, int64_t n,
                            int64_t vocab, int64_t width, int dtype, float scale, void *dtable,
                            void *workspace, size_t workspace_bytes, void *stream);

/* Layer norm of rows: u = x + residual, rounded to the type (residual NULL: u = x),
 * y = (u - mean u) / sqrt(mean (u - mean u)^2 + eps) * weight + bias (NULL: ones, zeros; both of type f32 if
 * weight_f32 != 0, else of the rows' type).  width <= 16384. */
typedef struct gear_hip_layer_norm_desc {
  const void *x, *residual;
  int64_t x_stride, residual_stride;
  int64_t rows, width;
  const void *weight, *bias;
  int32_t weight_f32, dtype;
  float eps;
} gear_hip_layer_norm_desc;
/* sum: u, with a residual; else NULL */
int gear_hip_layer_norm(const gear_hip_layer_norm_desc *desc, void *y, void *sum, void *stream);
/* Gradients from dy and (NULL: none) dsum, that of the sum: dx, which is the residual's as well, and of the weights
 * (of their type; NULL: not wanted).  desc->x is u, desc->residual is not looked at.
 * workspace, where a weight's gradient is wanted: gear_hip_layer_norm_backward_workspace_bytes(rows, width) bytes on
 * the device, 16-byte aligned. */
size_t gear_hip_layer_norm_backward_workspace_bytes(int64_t rows, int64_t width);
int gear_hip_layer_norm_backward(const gear_hip_layer_norm_desc *desc, const void *dy, int64_t dy_stride,
                                 const void *dsum, int64_t dsum_stride, void *dx, void *dweight, void *dbias,
                                 void *workspace, size_t workspace_bytes, void *stream);

/* Rows of logits; 0 < scale < 1e30, vocab <= 2^20, rows < 2^31 (gradients: rows * (vocab / 1024, rounded up) < 2^32).  z = scale * logits, lse = log sum_j exp z_j, p = exp(z - lse).
 * A logit of -inf is a token that is not allowed; rows that allow none (no logit of -1e30 or more, and no NaN) have lse = -inf,
 * log probabilities of -inf, entropy 0 and no gradient.  So the lowest numbers of f32 and bf16 are as good a mask; f16's, -65504, is a
 * logit like any other: a row of nothing else is a uniform distribution, and is masked with -inf instead.
 * NaN or +inf makes its row's results NaN. */
typedef struct gear_hip_logits_desc {
  const void *logits;
  int64_t row_stride, rows, vocab;
  int32_t dtype;
  float scale;
} gear_hip_logits_desc;
/* log_probs[i] = z[i][tokens[i]] - lse[i];  entropy[i] = -sum_j p_j log p_j;  the `top` (<= 64, <= vocab) largest logits
 * of a row, the lower token first among equals and NaN before all, as top_tokens and their log probabilities.  A row
 * whose token is none is not looked at: 0, 0, 0, and -1 with -inf.  tokens and log_probs may both be NULL.
 * workspace: gear_hip_token_log_probs_workspace_bytes(rows, vocab, top) bytes on the device, 256-byte aligned. */
size_t gear_hip_token_log_probs_workspace_bytes(int64_t rows, int64_t vocab, int64_t top);
int gear_hip_token_log_probs(const gear_hip_logits_desc *desc, const void *tokens, int tokens_i64, int64_t top,
                             float *log_probs, float *entropy, float *lse, float *top_log_probs,
                             int64_t *top_tokens, void *workspace, size_t workspace_bytes, void *stream);
/* dlogits = scale * (dlog_probs (1[j = token] - p_j) - dentropy p_j (log p_j + entropy)), in the logits' type, from the
 * forward call's lse and entropy.  dlog_probs, or dentropy and entropy, may be NULL. */
int gear_hip_token_log_probs_backward(const gear_hip_logits_desc *desc, const float *dlog_probs,
                                      const float *dentropy, const void *tokens, int tokens_i64, const float *lse,
                                      const float *entropy, void *dlogits, void *stream);
/* Divergence of rows from a teacher's `count` (<= 64) best tokens: q = softmax of top_logits over a row's entries
 * [rows][count] (entries without a token have no part), loss = sum_k q_k (log q_k - log p[top_tokens_k]).  Rows without
 * an entry are not looked at: 0.  A token that is named twice counts with both.
 * workspace: gear_hip_distill_workspace_bytes(rows, vocab) bytes on the device, 256-byte aligned. */
size_t gear_hip_distill_workspace_bytes(int64_t rows, int64_t vocab);
int gear_hip_distill(const gear_hip_logits_desc *desc, const void *top_tokens, int tokens_i64,
                     const float *top_logits, int64_t count, float *loss, float *lse, void *workspace,
                     size_t workspace_bytes, void *stream);
/* dlogits = scale * dloss (p_j - the q_k of entries that name j), from the forward call's lse. */
int gear_hip_distill_backward(const gear_hip_logits_desc *desc, const float *dloss, const void *top_tokens,
                              int tokens_i64, const float *top_logits, int64_t count, const float *lse,
                              void *dlogits, void *stream);

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif

#ifdef __cplusplus
}
#endif
#endif /* GEAR_HIP_H_ */
