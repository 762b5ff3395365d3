/*
 * fsgs.h — C-ABI of the MI355X-native Gaussian-splatting hot path (libfsgs.so).
 *
 * This is the drop-in boundary below FusionSense's gsplat operator surface.  The reference
 * reaches the same operations through gsplat 1.0.0's pybind11 module `gsplat.cuda._C`
 * (un-vendored; pinned at /root/reference/pyproject.toml:8) from two call sites:
 *     dn_splatter/dn_model.py:570-591   gsplat.rendering.rasterization(...)
 *     dn_splatter/dn_model.py:644-653   gsplat.rasterize_gaussians(...)   (legacy 0.1.x path)
 * and, for densify/prune statistics, nerfstudio's SplatfactoModel.after_train
 * (registered at dn_splatter/dn_model.py:1385-1389).
 *
 * Conventions (all entry points):
 *   - plain pointers to DEVICE memory + sizes; no torch types; fp32 / int32 / int64 only (the semantic
 *     head's operators also take bf16 / fp16, named by an FSGS_* element type)
 *   - all tensors contiguous, row-major, layouts as in the per-function comments
 *   - the caller owns every buffer (including scratch); the library never allocates
 *   - every call enqueues on `stream` (a hipStream_t passed as void*) and returns at once;
 *     the ONLY call that synchronises is fsgs_isect_count (it returns n_isects to the host,
 *     the same point at which the reference syncs)
 *   - return 0 on success, a negative FSGS_E* code otherwise; never throws; re-entrant
 *   - no global state: everything a launch depends on is an argument of the call (since round 4 that includes the
 *     dispatch order of the compositing backward and the lazy / idle-skipping switches of the per-Gaussian backward).
 *     The two process-wide setters of round 3 — fsgs_set_bwd_dispatch_stride, fsgs_set_lazy_sh_min_n — remain as
 *     DEPRECATED defaults that only a caller passing a negative value for the corresponding argument ever reads.
 *     The library reads NO environment variable (round 5): its A/B switches are build macros of csrc/ (make EXTRA=-D...)
 *   - FSGS_ABI_VERSION changes with every change of a signature or of a buffer's size / layout; a binding must refuse a
 *     library whose fsgs_abi_version() differs from the header it was written against (fusionsense_amd/_lib.py does)
 */
#ifndef FSGS_H
#define FSGS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef void *fsgs_stream_t; /* hipStream_t */

#define FSGS_OK 0
#define FSGS_EINVAL -1   /* bad argument (null pointer, unsupported size / channel count) */
#define FSGS_ELAUNCH -2  /* hipLaunch / runtime error; see fsgs_last_hip_error() */
#define FSGS_ESCRATCH -3 /* scratch arena too small */
#define FSGS_EPROTOCOL -4 /* a bounded cross-workgroup / host wait ran into its bound, or calls arrived out of order */

#define FSGS_ABI_VERSION 11
int fsgs_version(void);
int fsgs_abi_version(void); /* == FSGS_ABI_VERSION of the header the library was built from */
/* Lines of the packed gradient accumulator a caller that passes `replica_rows` > 0 must provide per Gaussian row:
 * `v_packed` is [fsgs_grad_replica_lines() * replica_rows, 16] floats, zeroed once (the last reader keeps it zeroed).
 * Gaussians of large 2-D footprint (det(cov2d) > 4096 px^4) spread their gradient atomics over these lines, picked
 * by tile and quadrant; `replica_rows` = 0 means one line per Gaussian and no spreading.  (No gsplat equivalent:
 * gsplat's rasterize_to_pixels_bwd adds into v_means2d / v_conics / v_colors / v_opacities directly.) */
int fsgs_grad_replica_lines(void);
const char *fsgs_error_string(int code);
int fsgs_last_hip_error(void); /* last hipError_t seen by this thread's failing call */

/* ---- E2: fully_fused_projection (gsplat._C.fully_fused_projection_fwd/bwd) ------------------
 * means[N,3] quats[N,4] (wxyz, normalised in-kernel) scales[N,3] viewmats[C,4,4] Ks[C,3,3]
 * -> radii[C,N] i32, means2d[C,N,2], depths[C,N], conics[C,N,3], compensations[C,N] (nullable).
 * Culled Gaussians get radii=0 and zeroed outputs. */
int fsgs_project_fwd(int C, int N, const float *means, const float *quats, const float *scales,
                     const float *viewmats, const float *Ks, int width, int height, float eps2d,
                     float near_plane, float far_plane, float radius_clip, int32_t *radii,
                     float *means2d, float *depths, float *conics, float *compensations,
                     fsgs_stream_t stream);

/* VJP of the above.  v_compensations nullable.  Writes (not accumulates) v_means[N,3],
 * v_quats[N,4], v_scales[N,3]; sums over cameras inside the kernel (deterministic).
 * v_viewmats[C,4,4] nullable; when given it is ACCUMULATED with atomics (zero it first). */
int fsgs_project_bwd(int C, int N, const float *means, const float *quats, const float *scales,
                     const float *viewmats, const float *Ks, int width, int height, float eps2d,
                     const int32_t *radii, const float *conics, const float *compensations,
                     const float *v_means2d, const float *v_depths, const float *v_conics,
                     const float *v_compensations, float *v_means, float *v_quats,
                     float *v_scales, float *v_viewmats, fsgs_stream_t stream);

/* ---- E3: spherical harmonics colour, fused with the rasterization() glue ---------------------
 * (gsplat._C.compute_sh_fwd/bwd + `dirs = means - campos`, `+0.5`, `clamp_min(0)` and the
 * depth-channel concat of render_mode "RGB+ED").
 * coeffs[N,K,3]; campos[C,3]; radii[C,N] mask; depths[C,N] (nullable -> no depth channel).
 * colors_out[C,N,D] with D = 3 (+1 if depths).  Gaussians with radii<=0 get rgb = 0.5. */
/* campos[C,3] = torch.inverse(viewmats)[:, :3, 3] for affine world-to-camera matrices. */
int fsgs_campos_from_viewmats(int C, const float *viewmats, float *campos, fsgs_stream_t stream);
int fsgs_sh_fwd(int C, int N, int K, int degree, const float *means, const float *campos,
                const float *coeffs, const int32_t *radii, const float *depths,
                float *colors_out, fsgs_stream_t stream);

/* v_colors[C,N,D] -> v_coeffs[N,K,3] (written; bases above `degree` get 0), v_means[N,3]
 * (ACCUMULATED into: the projection VJP has usually written it already), and
 * v_depths[C,N] (written, nullable; the pass-through gradient of the depth channel). */
int fsgs_sh_bwd(int C, int N, int K, int degree, const float *means, const float *campos,
                const float *coeffs, const int32_t *radii, int D, const float *v_colors,
                float *v_coeffs, float *v_means, float *v_depths, fsgs_stream_t stream);

/* Same kernels with the SH coefficients in FusionSense's stored split form
 * (gauss_params["features_dc"] [N,3] and ["features_rest"] [N,K-1,3], dn_model.py:294-304), which
 * saves the 2 x 192 B/Gaussian torch.cat at dn_model.py:543 and the split of its gradient. */
int fsgs_sh_fwd_split(int C, int N, int K, int degree, const float *means, const float *campos,
                      const float *features_dc, const float *features_rest, const int32_t *radii,
                      const float *depths, float *colors_out, fsgs_stream_t stream);
int fsgs_sh_bwd_split(int C, int N, int K, int degree, const float *means, const float *campos,
                      const float *features_dc, const float *features_rest, const int32_t *radii, int D,
                      const float *v_colors, float *v_features_dc, float *v_features_rest,
                      float *v_means, float *v_depths, int overwrite_means, int64_t replica_rows,
                      fsgs_stream_t stream);

/* fsgs_sh_fwd_split (one camera, with the depth channel) and fsgs_live_pack_normals in one launch: the colours go
 * straight into the packed per-Gaussian records [N,16] that the live-list kernels gather (no colour array is
 * written), normals_world [N,3] and the n_zero zeroed cells come out as from fsgs_live_pack_normals. */
int fsgs_sh_fwd_pack(int N, int K, int degree, const float *means, const float *campos, const float *features_dc,
                     const float *features_rest, const int32_t *radii, const float *depths, const float *means2d,
                     const float *conics, const float *opacities, const float *quats, const float *log_scales,
                     const float *c2w, float *packed, float *normals_world, float *zero_cells, int n_zero,
                     fsgs_stream_t stream);

/* Data-parallel training exchanges the FACTORS of the SH coefficient gradient instead of the gradient: per rank
 * and Gaussian the masked colour gradient (16 B) instead of 48 coefficient gradients (192 B), since
 * v_coeffs[n,k,:] = basis_k(dir(n)) * v_rgb[n,:].  fsgs_sh_bwd_colors = fsgs_sh_bwd_split for one camera without
 * the coefficient outputs: writes v_means and v_rgb_masked [N + 1,4] (rows 0..N-1: the colour gradient where the
 * clamp of `colors = max(SH + 0.5, 0)` is inactive and the Gaussian visible, else 0; row N: the camera centre).  fsgs_sh_coeff_grad rebuilds
 * scale * sum over R views; `gathered` = R blocks of (N + 1) x 4 floats: rows 0..N-1 = v_rgb_masked of view r,
 * row N = (camera centre, -).  Same replaced reference call as fsgs_sh_bwd. */
int fsgs_sh_bwd_colors(int N, int K, int degree, const float *means, const float *campos,
                       const float *features_dc, const float *features_rest, const int32_t *radii, int D,
                       const float *v_colors, float *v_rgb_masked, float *v_means, int overwrite_means, int64_t replica_rows,
                       fsgs_stream_t stream);
int fsgs_sh_coeff_grad(int R, int N, int K, int degree, const float *means, const float *gathered, float scale,
                       float *v_features_dc, float *v_features_rest, fsgs_stream_t stream);
/* fsgs_sh_coeff_grad and the Adam step of the two SH feature groups (as fsgs_adam_step would do it) in one launch:
 * the rebuilt mean gradient is applied as it leaves LDS and never written. */
int fsgs_sh_coeff_grad_adam(int R, int N, int K, int degree, const float *means, const float *gathered, float scale,
                            float *features_dc, float *exp_avg_dc, float *exp_avg_sq_dc, float lr_dc,
                            float *features_rest, float *exp_avg_rest, float *exp_avg_sq_rest, float lr_rest,
                            int step, double beta1, double beta2, float eps, fsgs_stream_t stream);
/* D = floats per v_colors row (its first three are the colour gradient): 3, 4 (then v_depths, if given,
 * receives column 3) or a wider stride, e.g. 16 for the rasterizer's packed gradient records.
 * overwrite_means != 0: v_means is written instead of accumulated into. */

/* ---- E4: isect_tiles (gsplat._C.isect_tiles), two passes --------------------------------------
 * Pass 1: tiles_per_gauss[C,N] i32 and its inclusive prefix sum cum_tiles[C,N] i64.
 * `legacy` != 0 selects the cuda_legacy bbox rule ((int)(c-r), (int)(c+r+1)) used by
 * gsplat.rasterize_gaussians.  Synchronises `stream` and stores the total in *n_isects_host.
 * n_rule_diff_host (nullable) receives the number of Gaussians whose tile rectangle differs
 * under the OTHER bbox rule; 0 means both rules bin this frame identically, so the legacy
 * normal pass may reuse the sorted lists of the RGB+ED pass.
 * scratch: fsgs_scan_scratch_bytes(C*N) bytes. */
size_t fsgs_scan_scratch_bytes(int64_t n);
int fsgs_isect_count(int C, int N, const float *means2d, const int32_t *radii, int tile_size,
                     int tile_width, int tile_height, int legacy, int32_t *tiles_per_gauss,
                     int64_t *cum_tiles, void *scratch, size_t scratch_bytes,
                     int64_t *n_isects_host, int64_t *n_rule_diff_host, fsgs_stream_t stream);

/* Pass 2: emit isect_ids[M] i64 = cam<<(32+tile_bits) | tile<<32 | bits(depth) and
 * flatten_ids[M] i32 = c*N+n, in (Gaussian, row-major tile) order. */
int fsgs_isect_emit(int C, int N, const float *means2d, const int32_t *radii, const float *depths,
                    const int64_t *cum_tiles, int tile_size, int tile_width, int tile_height,
                    int legacy, int64_t *isect_ids, int32_t *flatten_ids, fsgs_stream_t stream);

/* Live emission (tile_size 16; used by the fused get_outputs node, where gsplat's full lists are not
 * an output): a (Gaussian, tile) pair is counted / emitted only if the Gaussian can reach one of the
 * tile's 8x8 quadrants at alpha >= 1/255 (the same conservative test as fsgs_live_payload), and the
 * payload is  quadrant_mask << 28 | flatten_id  (C*N < 2^28).  tiles_per_gauss is still gsplat's
 * rectangle count.  Everything downstream (sort, offsets, prepare) then works on ~1/4 of the entries.
 * n_live_host: the live total, read back with a stream synchronisation; NULL = no read-back and no
 * synchronisation (the caller copies cum_live[C*N-1] itself and can overlap the wait with other work). */
int fsgs_isect_count_live(int C, int N, const float *means2d, const int32_t *radii, const float *conics,
                          const float *opacities, int tile_width, int tile_height,
                          int32_t *tiles_per_gauss, int32_t *live_per_gauss, int64_t *cum_live,
                          void *scratch, size_t scratch_bytes, int64_t *n_live_host, fsgs_stream_t stream);
int fsgs_isect_emit_live(int C, int N, const float *means2d, const int32_t *radii, const float *depths,
                         const float *conics, const float *opacities, const int64_t *cum_live,
                         int tile_width, int tile_height, int64_t *isect_ids, int32_t *payload,
                         fsgs_stream_t stream);

/* ---- E5: stable LSD radix sort of (i64 key, i32 value) pairs over key bits [0,end_bit) --------
 * Replaces cub::DeviceRadixSort::SortPairs.  Ping-pongs between (keys_a, vals_a) and
 * (keys_b, vals_b); returns 0 or 1 in *result_in_b to say where the sorted data ended up. */
size_t fsgs_sort_scratch_bytes(int64_t n);
int fsgs_sort_pairs(int64_t n, int64_t *keys_a, int32_t *vals_a, int64_t *keys_b, int32_t *vals_b,
                    int end_bit, void *scratch, size_t scratch_bytes, int *result_in_b,
                    fsgs_stream_t stream);

/* ---- E6: isect_offset_encode (gsplat._C.isect_offset_encode) ---------------------------------
 * offsets[C*n_tiles] i32: first sorted index of every (camera, tile). */
int fsgs_isect_offset_encode(int64_t n_isects, const int64_t *isect_ids_sorted, int C, int n_tiles,
                             int tile_bits, int32_t *offsets, fsgs_stream_t stream);

/* ---- E7 / E8: rasterize_to_pixels fwd/bwd (gsplat._C.rasterize_to_pixels_fwd/bwd and the
 * legacy rasterize_forward/backward).  D in {1,3,4}.  tile_size in [2,16].
 * means2d[C,N,2] conics[C,N,3] colors[C,N,D] opacities[C,N] backgrounds[C,D] (nullable)
 * -> render[C,H,W,D], alphas[C,H,W], last_ids[C,H,W] i32 (absolute index into flatten_ids). */
int fsgs_raster_fwd(int C, int N, int D, const float *means2d, const float *conics,
                    const float *colors, const float *opacities, const float *backgrounds,
                    int width, int height, int tile_size, int tile_width, int tile_height,
                    const int32_t *isect_offsets, const int32_t *flatten_ids, int64_t n_isects,
                    float *render, float *alphas, int32_t *last_ids, fsgs_stream_t stream);

/* Gradient outputs are ACCUMULATED with fp32 atomics: zero them first.
 * v_means2d_abs (the `absgrad` side output) nullable. */
int fsgs_raster_bwd(int C, int N, int D, const float *means2d, const float *conics,
                    const float *colors, const float *opacities, const float *backgrounds,
                    int width, int height, int tile_size, int tile_width, int tile_height,
                    const int32_t *isect_offsets, const int32_t *flatten_ids, int64_t n_isects,
                    const float *alphas, const int32_t *last_ids, const float *v_render,
                    const float *v_alphas, float *v_means2d, float *v_means2d_abs,
                    float *v_conics, float *v_colors, float *v_opacities, fsgs_stream_t stream);

/* ---- E7 / E8 fast path (tile_size == 16): "live lists" ----------------------------------------
 * (csrc/live.hip, raster_quad.hip, raster_live.hip; same reference functions as fsgs_raster_fwd/bwd:
 * gsplat 1.0.0 rasterize_to_pixels_{fwd,bwd} for dn_model.py:570-591 and the legacy
 * rasterize_forward/backward behind gsplat.rasterize_gaussians for dn_model.py:644-653.)
 * Every entry of the sorted tile lists carries an exact 4-bit mask of the tile's 8x8 quadrants the
 * Gaussian can reach at alpha >= 1/255.  A workgroup of four waves owns one quadrant: it reads the
 * tile's list itself, keeps the entries with its bit, gathers their 64-byte line from the packed
 * per-Gaussian table and composites 16 pixels x 4 consecutive records per step (quad prefix products
 * for the transmittance chain); the walked records are streamed out once for the segment-parallel
 * backward.  Results equal fsgs_raster_fwd/bwd on the raw lists; `meta` lists are untouched.
 *   packed   [C*N,16] f32 from fsgs_live_pack: {x,y,opacity,conic.a}{conic.b,conic.c,-,-}{colour[4]}{extra[3],-}
 *   payload  [M] i32: (quadrant mask << 28) | flatten id — what fsgs_isect_emit_live writes, or
 *            fsgs_live_payload from plain lists (so C*N < 2^28)
 *   records  4 * fsgs_quad_stream_capacity(...) * (render_extra ? 16 : 12) floats, n_rec [4, C*th*tw] i32:
 *            the walked part of every quadrant's list, written for fsgs_raster_bwd_quad (both nullable
 *            together for inference).  Record = {x,y,opacity,conic.a} {conic.b,conic.c,bits(list index),
 *            bits(flatten id)} {colour, zero padded} [{extra xyz,-}]
 *   seg_state (nullable for inference) 4 * fsgs_quad_seg_slots(...) * 64 * (1+D+E) floats: every pixel's
 *            (T, accumulated colour) after each 64-record segment of its quadrant's stream, so that the
 *            backward can process segments independently
 *   render_extra [C,H,W,3] (nullable, D == 4): a second per-Gaussian 3-vector (FusionSense's camera-space
 *            normals, the 4th float4 of the packed line) composited in the SAME walk over a background of
 *            ones — what gsplat.rasterize_gaussians returns for it; E = 3 then, else 0
 *   max_last [fsgs_raster_quad_max_cells()] (nullable): partial maxima of the last output channel, raised
 *            with atomics — zero them first (fsgs_live_pack does); feed fsgs_epilogue_fwd with
 *            n_partial = -fsgs_raster_quad_max_cells() (dn_model.py:611-613 fills empty depth pixels with
 *            the image maximum)
 *   normalize_last != 0 implements render_mode "ED"/"RGB+ED" in-kernel: the last channel leaves as
 *            accumulated / max(alpha, 1e-10) (gsplat does this with three torch ops after the kernel), and
 *            the backward expects v_render's last channel to be the gradient of that normalised value.
 *   v_packed [C*N,16] f32, ACCUMULATED with atomics (zero it first): per (camera, Gaussian)
 *            [0..3] v_colors [4..6] v_conics [7..8] v_means2d [9..10] v_means2d_abs [11] v_opacities
 *            [12..14] v_extra.  The extra plane's gradient reaches conics / opacities / its own colours but
 *            NOT v_means2d / v_means2d_abs (the reference detaches xys for that pass, dn_model.py:638). */
int fsgs_raster_quad_max_cells(void);
int64_t fsgs_quad_stream_capacity(int C, int tile_width, int tile_height, int64_t n_isects);
int64_t fsgs_quad_seg_slots(int C, int tile_width, int tile_height, int64_t n_isects);
int fsgs_live_pack(int D, int64_t n_gauss_total, const float *means2d, const float *conics,
                   const float *colors, const float *opacities, const float *extra, float *packed,
                   float *zero_cells /* nullable: n_zero floats set to 0 */, int n_zero, fsgs_stream_t stream);
/* fsgs_live_pack (D = 4) whose extra plane is the camera-space normal of every Gaussian, computed in the
 * same launch instead of by fsgs_normals_fwd; normals_world [N,3] is the side output (single camera). */
int fsgs_live_pack_normals(int64_t N, const float *means2d, const float *conics, const float *colors,
                           const float *opacities, const float *quats, const float *log_scales,
                           const float *means, const float *c2w, float *packed, float *normals_world,
                           float *zero_cells, int n_zero, fsgs_stream_t stream);
int fsgs_live_payload(const int64_t *isect_ids, const int32_t *flatten_ids, int64_t n_isects,
                      const float *packed, int64_t n_gauss_total, int tile_width, int tile_bits,
                      int32_t *payload, fsgs_stream_t stream);
int fsgs_raster_fwd_quad(int C, int D, const float *packed, const int32_t *payload,
                         const int32_t *isect_offsets, int64_t n_isects, const float *backgrounds,
                         int width, int height, int tile_width, int tile_height, int normalize_last,
                         float *render, float *alphas, int32_t *last_ids, float *records, int32_t *n_rec,
                         float *seg_state, float *render_extra, float *max_last,
                         int32_t *tile_open /* nullable [C*th*tw]: see fsgs_tile_zcut_update */,
                         int walk /* FSGS_WALK_*: how THIS launch walks the lists */,
                         void *tail_scratch /* nullable */, int64_t tail_scratch_bytes, int tail_items,
                         int handoff_records, int handoff_rel_len, const int32_t *handoff_gate /* nullable */,
                         int64_t tail_epoch, int32_t *seg_split /* nullable */,
                         int32_t *bwd_queue /* nullable */, int bwd_queue_items,
                         const int32_t *tile_order /* nullable; FSGS_WALK_ONE_WAVE, C == 1: the tiles longest list first
                         (fsgs_project_bin_live_fill_sh_pack) — the quadrants are then walked once, in that order,
                         instead of in two passes (tiles above twice the mean list length, then the others) */,
                         fsgs_stream_t stream);
/* Long streams in the backward (round 5): seg_split [4, C*th*tw] i32 (next to n_rec) receives, per quadrant, the first
 * 64-record segment its own backward workgroup walks — 0 unless the stream has more than 8 segments AND bwd_queue
 * ([4 + 4 * bwd_queue_items] i32: a counter the CALLER ZEROES before the call + 3 pad words, then int4 items) had room:
 * then the segments in front of the last 8 are queued in groups of 8 for extra workgroups of fsgs_raster_bwd_quad* (pass
 * it the same three arguments).  A list of 44 segments (config #3's hull tiles) is then walked by six workgroups side
 * by side instead of 11 rounds of one.  Gradients are unchanged up to the order of the float atomics. */
/* Dispatch order of the backward (round 5): bwd_order (nullable; needs bwd_queue, C == 1) = [32, 4 * th * tw] i32, filled
 * between the forward and the backward by fsgs_epilogue_fwd_order (below): every quadrant is filed under a class of its
 * own share's record count (2^order_shift records wide, the last class open-ended), bwd_order[class][slot] = the quadrant's position
 * in the backward's grid; the classes' 32 i32 counters sit BEHIND the queue's items (bwd_queue then needs 4 + 4 *
 * bwd_queue_items + 32 words, zeroed by the caller).  fsgs_raster_bwd_quad* given bwd_order start the quadrants longest
 * class first (dispatch_stride is then not used): a backward workgroup's time is its quadrant's share, and the launch
 * ends with its last round of workgroups — config #3's trained scene 0.191 -> 0.174 ms.  Gradients are unchanged up to
 * the order of the float atomics. */
/* Hand-off of long walks (round 5; FSGS_WALK_ONE_WAVE, handoff_records > 0): a wave that has streamed `handoff_records`
 * records and still has open pixels and list entries left stops at the end of its 64-entry chunk and queues the rest of
 * its list; TAIL workgroups of the same launch (one wave per queued 64-entry chunk; `tail_items` of them are launched,
 * which the caller sizes from the demand counter of earlier frames) form every chunk's transmittance factor independently, takes the transmittance at its start from its predecessors' factors, composites the chunk with
 * the reference's stop rule and adds the chunks' partial sums in list order — a list of n entries costs two chunk walks
 * of latency instead of n dependent steps (config #3 after densification: lists of 2 800 entries).  Same outputs up to
 * the association of products and sums per chunk (image tolerance), bit-reproducible, same streams / segment states /
 * n_rec for the backward.  `tail_scratch`: fsgs_raster_fwd_tail_scratch_bytes(max_items) bytes, ZEROED ONCE by the
 * caller and then only ever passed to this function; `tail_epoch` >= 1 must increase by one with every call that passes
 * the scratch (two frames' counters alternate inside it).  A queue that runs full makes the remaining walks finish
 * serially (exact, only slower).  handoff_records = 0: the plain one-wave walk (tail_scratch may be NULL).
 * fsgs_raster_fwd_tail_error: 1 if any look-back wait ever ran into its bound (never observed; results of that frame
 * are then invalid), 0 otherwise — a synchronous read for tests. */
int64_t fsgs_raster_fwd_tail_scratch_bytes(int max_items);
int fsgs_raster_fwd_tail_error(const void *tail_scratch, fsgs_stream_t stream);
/* walk (fsgs_raster_fwd_quad): FSGS_WALK_FOUR_WAVES — a workgroup of four waves per 8x8 quadrant, lane = (pixel, one of
 * four consecutive records); FSGS_WALK_ONE_WAVE (render_extra != NULL only; FSGS_EINVAL otherwise) — one wave per quadrant,
 * lane = pixel, one record per step: half the vector instructions per (quadrant, record), but a quadrant's walk is one
 * wave's dependent chain (~0.17 us per record on MI355X), so the frame's longest list bounds the launch unless long
 * walks are handed off (handoff_records, below).  Same images up
 * to the association of the transmittance products (<= 1 ulp per step), same streams for the backward (the one-wave
 * walk writes no padding records).  Without the hand-off which is faster depends on the frame (config #2: 95 vs 79 us;
 * config #3 after densification, lists of 2 800 entries: 153 vs 278 us); with it the one-wave walk wins on both (78 /
 * 100 us) and fusionsense_amd/fused.py uses it for every frame. */
#define FSGS_WALK_FOUR_WAVES 0
#define FSGS_WALK_ONE_WAVE 1
int fsgs_raster_bwd_quad(int C, int D, const float *records, const int32_t *n_rec,
                         const int32_t *isect_offsets, int64_t n_isects, const float *backgrounds,
                         int width, int height, int tile_width, int tile_height, int normalize_last,
                         const float *render, const float *alphas, const int32_t *last_ids,
                         const float *v_render, const float *v_alphas, const float *seg_state,
                         int with_abs, const float *render_extra, const float *v_render_extra,
                         float *v_packed, int dispatch_stride, const int32_t *seg_split /* nullable */,
                         const int32_t *bwd_queue /* nullable; C == 1 */, int bwd_queue_items,
                         const int32_t *bwd_order /* nullable */, fsgs_stream_t stream);
/* dispatch_stride (fsgs_raster_bwd_quad, fsgs_raster_bwd_quad_images) — the dispatch order of THIS launch's quadrants:
 * 0 or 1 = row-major, k > 1 = consecutive workgroups take quadrants k apart (raised to the next value coprime with the
 * number of quadrants).  Same gradients up to the order of the float atomics; which order is faster depends on the scene
 * (neighbouring quadrants share Gaussians and collide on their gradient lines; far-apart ones lose the L2 residency of
 * those lines): fusionsense_amd/fused.py goes by the frame's size (7 apart up to 2^20 pixels, row-major above; measured
 * 0.169 vs 0.176 ms at 800x800, 0.927 vs 0.947 ms at 1080p the other way round).  A launch argument since round 4: no
 * state outlives the call.  DEPRECATED: a negative value takes the process-wide default that
 * fsgs_set_bwd_dispatch_stride sets (initially env FSGS_BWD_PERM or 0; returns the previous value) — round-3 callers. */
int fsgs_set_bwd_dispatch_stride(int stride);

/* fsgs_epilogue_bwd + fsgs_raster_bwd_quad for FusionSense's get_outputs (one camera; RGB + expected depth and the
 * normal plane in one walk): takes the gradients of the rgb / depth / normal images (and of the accumulation,
 * nullable) and derives v_render / v_alphas / v_render_extra per pixel inside the kernel
 * (/root/reference/dn_splatter/dn_model.py:602-613, 655-664).  background: 3 floats. */
int fsgs_raster_bwd_quad_images(const float *records, const int32_t *n_rec, const int32_t *isect_offsets,
                                int64_t n_isects, int width, int height, int tile_width, int tile_height,
                                const float *render, const float *alphas, const int32_t *last_ids,
                                const float *render_extra, const float *background, const float *v_rgb,
                                const float *v_depth, const float *v_normal, const float *v_alpha_in,
                                const float *seg_state, int with_abs, float *v_packed, int64_t replica_rows,
                                int dispatch_stride, const int32_t *seg_split /* nullable */,
                                const int32_t *bwd_queue /* nullable */, int bwd_queue_items,
                                const int32_t *bwd_order /* nullable */, fsgs_stream_t stream);
/* replica_rows (here and in fsgs_gaussian_bwd; 0 = off): Gaussians with a large 2-D footprint (det(conic) < 1/4096)
 * own FOUR gradient lines, replica_rows rows apart in v_packed ([4 * replica_rows, 16], zeroed): the compositing
 * backward picks the replica from the tile and the 8x8 quadrant, so that the hundreds of workgroups a large Gaussian
 * is seen from do not serialise on one 64-byte line.  The SH backward (fsgs_sh_bwd_split / _h16 / fsgs_sh_bwd_colors
 * with D = 16 and replica_rows > 0) sums the replicas' colour gradients of every Gaussian of radius >= 24 px (a
 * superset: unwritten replicas hold zeros) as it reads them; fsgs_gaussian_bwd, the last reader, folds and clears
 * all of them. */
/* ---- Sort + offsets for live lists as a partition by tile plus a sort inside every tile's bucket
 * (same results, bit for bit, as fsgs_sort_pairs on the key bits + fsgs_isect_offset_encode; replaces
 * the same reference calls).  isect_ids [n] are the UNSORTED keys cam|tile|depth-bits of
 * fsgs_isect_emit_live, payload [n] = quadrant mask << 28 | flatten id.  Outputs: isect_offsets
 * [C*th*tw + 1] (last entry = n), payload_sorted [n], isect_ids_sorted [n] (nullable).
 * C*th*tw <= fsgs_tile_sort_max_tiles().  Any bucket size is handled (LDS up to 8192 entries per tile,
 * in place beyond that: slow — use fsgs_sort_pairs when tiles are that dense). */
int fsgs_tile_sort_max_tiles(void);
size_t fsgs_tile_sort_scratch_bytes(int64_t n, int n_tiles_total);
int fsgs_tile_sort(int64_t n, const int64_t *isect_ids, const int32_t *payload, int C, int tile_width,
                   int tile_height, int32_t *isect_offsets, int32_t *payload_sorted,
                   int64_t *isect_ids_sorted, void *scratch, size_t scratch_bytes, fsgs_stream_t stream);

/* ---- Direct binning of the live pairs: fsgs_isect_count_live + fsgs_isect_emit_live + fsgs_tile_sort as two
 * calls that never write the pairs in emission order (same outputs, bit for bit; replaces gsplat 1.0.0
 * `isect_tiles(sort=True)` + `isect_offset_encode` as reached from
 * /root/reference/dn_splatter/dn_model.py:570-591, for tile 16).
 *   fsgs_bin_live_count: enumerates the (Gaussian, tile) pairs, counts the live ones per tile and scans:
 *       tiles_per_gauss [C,N] (gsplat's count, nullable), isect_offsets [C*th*tw + 1] with the last entry =
 *       the number of live pairs (copy it to the host to size the second call's buffers).
 *   fsgs_bin_live_emit: enumerates again, drops every live pair into its tile's bucket and sorts the
 *       buckets on (depth, flatten id): payload_sorted [n_live] = quadrant mask << 28 | flatten id.
 * n_live_mapped (nullable): a DEVICE-ACCESSIBLE HOST pointer to FOUR ints (mapped pinned memory): [0] receives the
 * number of live pairs, then [1] is set to 1 (system-scope release) by the last kernel of the call: a caller that
 * cleared [1] beforehand can poll it instead of waiting for the stream; no copy launch.  [2] (input, 0 = none) is a
 * CAPACITY: every entry of isect_offsets, the last one included, is clamped to it, while [0] still receives the
 * true total.  A caller that sizes the second call's buffers from an estimate (n_live := the capacity, for
 * fsgs_bin_live_emit and the kernels after it; fsgs_raster_fwd_quad with n_isects = -capacity) therefore needs no
 * host wait between the two calls, stays inside its buffers whatever the frame holds, and finds out from
 * [0] > [2] — whenever it next looks — that the lists were truncated and the frame must be redone.  [3] reserved.
 * table_scratch: fsgs_bin_live_table_bytes(C, N, tw, th) bytes, untouched between the two calls;
 * buckets: n_live 64-bit words.  C*th*tw <= fsgs_bin_live_max_tiles(). */
int fsgs_bin_live_max_tiles(void);
size_t fsgs_bin_live_table_bytes(int C, int N, int tile_width, int tile_height);
int fsgs_bin_live_count(int C, int N, const float *means2d, const int32_t *radii, const float *conics,
                        const float *opacities, int tile_width, int tile_height, int32_t *tiles_per_gauss,
                        int32_t *isect_offsets, void *table_scratch, size_t table_bytes, int32_t *n_live_mapped,
                        fsgs_stream_t stream);
/* fsgs_project_fwd_act (one camera) + fsgs_bin_live_count as one call: the count pass projects its Gaussians itself
 * (same statements, csrc/project_math.h) and writes the projection's outputs for the later passes. */
int fsgs_project_bin_live_count(int N, const float *means, const float *quats, const float *log_scales,
                                float *opac_logit, int binarise, float binary_threshold, const float *viewmat,
                                const float *K, int width, int height, float eps2d, float near_plane, float far_plane,
                                float radius_clip, float *scales_out, float *opac_out, int32_t *radii, float *means2d,
                                float *depths, float *conics, int tile_width, int tile_height,
                                int32_t *tiles_per_gauss, int32_t *isect_offsets, void *table_scratch,
                                size_t table_bytes, int32_t *n_live_mapped, fsgs_stream_t stream);
/* An Adam step over up to 8 tensors, as an argument block (the arrays of fsgs_adam_step_h16). */
typedef struct fsgs_adam_groups {
    int n_groups;
    float *params[8];
    const float *grads[8];
    float *exp_avg[8];
    float *exp_avg_sq[8];
    void *half_mirror[8]; /* nullable entries */
    int64_t numel[8];
    float lr[8];
    int step;
    double beta1, beta2;
    float eps;
} fsgs_adam_groups;

/* fsgs_project_bin_live_count with independent work riding in its launches (same outputs as the separate calls):
 *  - packed != NULL: fsgs_sh_fwd_pack (16 stored coefficients, split features; opacities = opac_out, the other
 *    shared arrays as named) runs in the launch of the count pass's table scan — a few hundred latency-bound
 *    workgroups scan while the rest of the machine evaluates colours and packs records;
 *  - adam != NULL: that Adam step (fsgs_adam_step_h16 semantics) runs in the launch of the count pass itself.  None
 *    of its tensors may be an input of the count pass (means, quats, log_scales, opacity logits): it is meant for
 *    the SH features' update of the previous iteration, which the colours of this one (above) then see.
 *  - tile_zcut != NULL (occlusion cut, one float per tile, +inf = none): a pair whose Gaussian lies behind its tile's
 *    cut depth is neither counted here nor binned by fsgs_bin_live_emit(_split), which must be given the SAME array;
 *    the cuts come from fsgs_tile_zcut_update of an earlier frame of the same view, which also validates this frame.
 *    A Gaussian behind the largest cut of every 4x4-tile block its rectangle touches is dropped before the pair loop.
 *  - kept != NULL ([N] bytes, written): kept[n] = 1 if Gaussian n has at least one binned pair (live and not behind a
 *    cut), else 0.  A Gaussian with kept = 0 is in no tile's list, so the riding SH forward neither reads its
 *    coefficients nor writes its packed record (the record is never gathered); normals_world is written for all.
 *    Meant for dense scenes, where most Gaussians are in no list; it makes the coefficient loads dependent ones.
 * _h16: quats / log_scales / opacity logits / features are IEEE-half mirrors (as in fsgs_project_bin_live_count_h16
 * and fsgs_sh_fwd_pack_h16). */
int fsgs_project_bin_live_count_sh_pack(
    int N, const float *means, const float *quats, const float *log_scales, float *opac_logit, int binarise,
    float binary_threshold, const float *viewmat, const float *K, int width, int height, float eps2d, float near_plane,
    float far_plane, float radius_clip, float *scales_out, float *opac_out, int32_t *radii, float *means2d,
    float *depths, float *conics, int tile_width, int tile_height, int32_t *tiles_per_gauss, int32_t *isect_offsets,
    void *table_scratch, size_t table_bytes, int32_t *n_live_mapped, int degree, const float *campos,
    const float *features_dc, const float *features_rest, const float *c2w, float *packed, float *normals_world,
    float *zero_cells, int n_zero, const fsgs_adam_groups *adam, const float *tile_zcut, uint8_t *kept,
    int32_t *tile_order /* nullable [tw * th]: the tiles longest list first (as from ..._fill_sh_pack; packed != NULL) */,
    fsgs_stream_t stream);
int fsgs_project_bin_live_count_sh_pack_h16(
    int N, const float *means, const void *quats_h, const void *log_scales_h, void *opac_logit_h,
    float *opac_logit_master, int binarise, float binary_threshold, const float *viewmat, const float *K, int width,
    int height, float eps2d, float near_plane, float far_plane, float radius_clip, float *scales_out, float *opac_out,
    int32_t *radii, float *means2d, float *depths, float *conics, int tile_width, int tile_height,
    int32_t *tiles_per_gauss, int32_t *isect_offsets, void *table_scratch, size_t table_bytes, int32_t *n_live_mapped,
    int degree, const float *campos, const void *features_dc_h, const void *features_rest_h, const float *c2w,
    float *packed, float *normals_world, float *zero_cells, int n_zero, const fsgs_adam_groups *adam,
    const float *tile_zcut, uint8_t *kept, int32_t *tile_order /* nullable */, fsgs_stream_t stream);
int fsgs_bin_live_emit(int C, int N, const float *means2d, const int32_t *radii, const float *depths,
                       const float *conics, const float *opacities, int tile_width, int tile_height,
                       const int32_t *isect_offsets, const void *table_scratch, int64_t n_live, void *buckets,
                       int32_t *payload_sorted, const float *tile_zcut /* nullable; C == 1 */,
                       int32_t *long_flag /* nullable */, int rel_gate, fsgs_stream_t stream);
/* ---- Count-free binning (round 5): ONE enumeration of the (Gaussian, tile) pairs instead of two.  Replaces, for a view
 * whose previous frame told how much room every tile's bucket needs, the chain fsgs_project_bin_live_count_sh_pack ->
 * fsgs_bin_live_emit (same outputs, lists bit for bit; the same reference calls: gsplat 1.0.0 fully_fused_projection +
 * isect_tiles(sort=True) + isect_offset_encode + spherical_harmonics as reached from dn_model.py:570-591).
 *   bucket_base [T + 1] i32: tile t's bucket is words bucket_base[t] .. bucket_base[t + 1] of `buckets` (bucket_words
 *       >= bucket_base[T] 64-bit words); tile_cursor [T] i32, ZERO on entry and zero again on return;
 *   outputs beside the projection's and the packing's: tiles_per_gauss, isect_offsets [T + 1] (exact and compact; the
 *       last entry = the number of live pairs, clamped to n_live_mapped[2] like fsgs_bin_live_count's),
 *       next_bucket_base [T + 1] = exclusive sums of (int)(count * growth) + slack: the room for this view's NEXT frame;
 *   n_live_mapped (device-accessible host int[4], as for fsgs_bin_live_count): [0] the total, [3] = 1 if some tile
 *       outgrew its bucket — its surplus pairs were dropped and the caller must redo the frame through the two-pass
 *       route before anything with side effects has consumed the lists — then [1] = 1.
 * One camera, fp32 attributes, degree <= 3 with 16 stored coefficients, no occlusion cuts, N <= 1024 x 65535.
 * fsgs_bin_live_sort_buckets: the in-tile sorts, bucket t -> payload_sorted[isect_offsets[t] ..). */
int fsgs_project_bin_live_fill_sh_pack(
    int N, const float *means, const float *quats, const float *log_scales, float *opac_logit, int binarise,
    float binary_threshold, const float *viewmat, const float *K, int width, int height, float eps2d, float near_plane,
    float far_plane, float radius_clip, float *scales_out, float *opac_out, int32_t *radii, float *means2d,
    float *depths, float *conics, int tile_width, int tile_height, int32_t *tiles_per_gauss, int32_t *isect_offsets,
    const int32_t *bucket_base, int32_t *tile_cursor, void *buckets, int64_t bucket_words, int32_t *next_bucket_base,
    float growth, int slack, int32_t *n_live_mapped, int degree, const float *campos, const float *features_dc,
    const float *features_rest, const float *c2w, float *packed, float *normals_world, float *zero_cells, int n_zero,
    int32_t *tile_order /* nullable */, fsgs_stream_t stream);
int fsgs_bin_live_sort_buckets(int tile_width, int tile_height, const int32_t *isect_offsets,
                               const int32_t *bucket_base, void *buckets, int32_t *payload_sorted,
                               int32_t *long_flag /* nullable */, int rel_gate, const int32_t *tile_order /* nullable */,
                               fsgs_stream_t stream);
/* tile_order [tw * th] i32 (nullable): the bookkeeping workgroup of fsgs_project_bin_live_fill_sh_pack leaves the tiles
 * longest list first (classes of 64 entries) there, and fsgs_bin_live_sort_buckets dispatches its workgroups in that order:
 * a tile's sort takes as long as its list is long, and the launch is 5-7 rounds of resident workgroups. */
/* long_flag (round 5; a word the caller zeroes): set to 1 if any tile's list is longer than rel_gate times the mean list
 * length — the frame statistic fsgs_raster_fwd_quad's hand-off is gated on (handoff_gate): only frames that HAVE lists far
 * beyond the bulk (config #3's hull tiles: 16 x the mean; config #2's longest list: 5.7 x) queue anything. */

/* fsgs_bin_live_emit for buckets of any size: tiles with more than 1024 live pairs are first split into depth
 * slabs of ~512 (monotone in depth, so sorted slabs in order = a sorted tile), every slab sorted like a small
 * tile.  Same outputs, bit for bit; one more pass over the 64-bit words instead of the six radix passes that
 * scenes with thousands of pairs per tile otherwise need.  buckets, buckets2: n_live words each. */
size_t fsgs_bin_live_split_scratch_bytes(int C, int tile_width, int tile_height, int64_t n_live);
int fsgs_bin_live_emit_split(int C, int N, const float *means2d, const int32_t *radii, const float *depths,
                             const float *conics, const float *opacities, int tile_width, int tile_height,
                             const int32_t *isect_offsets, const void *table_scratch, int64_t n_live, void *buckets,
                             void *buckets2, void *split_scratch, size_t split_bytes, int32_t *payload_sorted,
                             const float *tile_zcut /* nullable; C == 1 */, fsgs_stream_t stream);

/* Occlusion cut (no gsplat equivalent; an exact speculation on temporal coherence).  A dense scene's tiles turn opaque
 * after a small depth prefix of their sorted lists (BASELINE config #4: 2 % of 39 M live pairs are ever composited), yet
 * every pair is reach-tested twice, binned and sorted.  A trainer that revisits its views hands the two binning passes a
 * per-tile cut depth taken from the view's previous frame: pairs behind it are not binned.  The kept pairs are a depth
 * PREFIX of the tile's full list, so a frame in which every cut tile saturates inside its prefix is bit-identical to the
 * uncut frame — images, last_ids, record streams, gradients; any other frame must be redone without cuts.
 * fsgs_raster_fwd_quad(tile_open != NULL) marks the tiles in which a pixel was still transparent at the end of its list;
 * this call (one camera) turns that and last_ids into
 *   zcut_out[t] = +inf if tile t was open — or saturated only within the last tail_frac of its list (such a tile gains
 *                 little from a cut and is the one found open a visit later; tail_frac, 0.25 in the trainer) —, else
 *                 depth(deepest composited entry of t) + max(margin_span * (that depth - the tile's first entry's
 *                 depth), margin_rel * that depth),
 *   zcut_cand[t]      = 1 for every open tile that had been binned with a finite zcut_in (the "candidates"),
 *   verdict_mapped[0] = 2 if there is a candidate, else 0 (the frame is exact), and
 *   verdict_mapped[1] = 1 once [0] has landed (host-mapped memory; the caller clears [1] beforehand);
 * tile_open is left cleared, bad_scratch (one zeroed int32 on the device) is left zeroed.  zcut_cand ([T] int32, zeroed)
 * is required with zcut_in.  After a verdict of 2 the caller runs fsgs_tile_zcut_recheck: an open tile under a cut
 * spoils the frame only if a LIVE pair of it lies behind the cut (a tile that barely saturated one visit ago and does
 * not now has usually lost nothing); verdict_mapped[0] = 1 there means the frame is INVALID.  The recheck applies the
 * binning's reach test to the candidate tiles only (one thread per Gaussian over its gsplat rectangle) and leaves
 * zcut_cand zeroed. */
int fsgs_tile_zcut_update(int tile_width, int tile_height, int width, int height, const int32_t *last_ids,
                          const int32_t *payload, const float *depths, const int32_t *isect_offsets,
                          int32_t *tile_open, const float *zcut_in, int32_t *zcut_cand, float *zcut_out,
                          int32_t *bad_scratch, int32_t *verdict_mapped, float margin_span, float margin_rel,
                          float tail_frac, fsgs_stream_t stream);
int fsgs_tile_zcut_recheck(int N, const float *means2d, const int32_t *radii, const float *depths, const float *conics,
                           const float *opacities, int tile_width, int tile_height, const float *zcut_in,
                           int32_t *zcut_cand, int32_t *bad_scratch, int32_t *verdict_mapped, fsgs_stream_t stream);


/* Split packed gradient records into the five gsplat-shaped arrays (written, not accumulated).
 * rezero != 0: v_packed is cleared after it has been read, ready for the next frame's atomics. */
int fsgs_raster_unpack_grads(int64_t total, int D, float *v_packed, int rezero, float *v_means2d,
                             float *v_means2d_abs, float *v_conics, float *v_colors,
                             float *v_opacities, float *v_extra, float *v_last, fsgs_stream_t stream);
/* v_extra[C*N,3] and v_last[C*N] (the last colour channel's gradient, i.e. v_depths when the depth
 * channel rides in colours) are optional outputs. */

/* ---- a-11: per-Gaussian normals (dn_splatter/dn_model.py:618-636 as one kernel) ---------------
 * quats[N,4] (any norm), log_scales[N,3], means[N,3], c2w[3,4] (OpenGL) ->
 * normals_world[N,3] (what the reference stores in gauss_params["normals"]),
 * normals_cam[N,3] = n @ c2w[:3,:3]. */
int fsgs_normals_fwd(int N, const float *quats, const float *log_scales, const float *means,
                     const float *c2w, float *normals_world, float *normals_cam,
                     fsgs_stream_t stream);
/* v_normals_cam[N,3] -> v_quats[N,4] (written). */
int fsgs_normals_bwd(int N, const float *quats, const float *log_scales, const float *means,
                     const float *c2w, const float *v_normals_cam, float *v_quats,
                     fsgs_stream_t stream);

/* ---- a-12: SplatfactoModel.after_train statistics in one pass ----------------------------------
 * vis = radii>0: vis_counts += 1; xys_grad_norm += ||absgrad||_2; max_2Dsize = max(., radii/max(H,W)) */
int fsgs_densify_stats(int N, const int32_t *radii, const float *absgrad, float inv_max_hw,
                       float *xys_grad_norm, float *vis_counts, float *max_2Dsize,
                       fsgs_stream_t stream);

/* ---- a-13: densify/prune row movement -----------------------------------------------------------
 * Order-preserving stream compaction of row-major [n_rows, row_floats] fp32 tensors by a
 * byte mask (keep[i] != 0).  fsgs_mask_scan builds positions once (exclusive scan of keep,
 * i64) and returns nothing to the host; fsgs_compact_rows applies them to one tensor. */
int fsgs_mask_scan(int64_t n_rows, const uint8_t *keep, int64_t *positions, void *scratch,
                   size_t scratch_bytes, fsgs_stream_t stream);
int fsgs_compact_rows(int64_t n_rows, int row_floats, const uint8_t *keep,
                      const int64_t *positions, const float *src, float *dst,
                      fsgs_stream_t stream);
/* fsgs_compact_rows for n_jobs <= 32 tensors in one launch: job j moves the kept rows of src[j] ([n_rows[j], row_floats[j]])
 * to dst[j] + positions[j][row] * row_floats[j] under its own mask keep[j].  The six arrays are HOST arrays of n_jobs
 * entries (their elements device pointers); jobs of zero rows are skipped. */
int fsgs_compact_rows_multi(int n_jobs, const int64_t *n_rows, const int *row_floats, const uint8_t *const *keep,
                            const int64_t *const *positions, const float *const *src, float *const *dst,
                            fsgs_stream_t stream);
/* a-14: out_mask[i] = 1 when point i [n,3] lies inside ANY of n_boxes oriented boxes, 0 otherwise.  A box is 18 floats:
 * centre (3), three unit axes (3 x 3, one per row), lower (3) and upper (3) bounds of the box's extent along the axes;
 * inside = lower <= (p - centre) . axis <= upper on all three axes, bounds inclusive.  Replaces the per-patch
 * points_in_non_aabb loop of touch_pruning / add_touch_patch (dn_splatter/dn_model.py:1173-1184, 1284-1294, 1996-2034). */
int fsgs_points_in_boxes(int64_t n, const float *points, int n_boxes, const float *boxes, uint8_t *out_mask,
                         fsgs_stream_t stream);
/* a-14: for every query [nq,3] the nearest of points [np,3] (np >= 1): Euclidean distance (out_dist, nullable) and
 * index (out_idx, REQUIRED since ABI 7: the point set is sliced over workgroups, which meet in out_idx's 64-bit words;
 * lowest index on ties; all zeros with want_idx == 0, which saves the kernel its index bookkeeping).  active (nullable,
 * [nq] bytes): queries whose byte is 0 are skipped — distance +inf, index 0.  Replaces torch.cdist(...).min(-1) in
 * hull_pruning (dn_splatter/dn_model.py:1258-1264) and the k=1 neighbour search of add_touch_patch (:1181-1182). */
int fsgs_nearest_point(int nq, const float *queries, int np, const float *points, const uint8_t *active, float *out_dist,
                       int64_t *out_idx, int want_idx, fsgs_stream_t stream);
/* The same search for fsgs_refine_mark (ABI 10): out_words [nq] keeps the workgroups' raw 64-bit words (squared-distance
 * bits above index bits, ~0 = no point compared) — no unpacking launch —, and the queries that matter are chosen in the
 * launch: those within `close_radius` of `center` (3 floats, HOST memory; hull_pruning's ``norm(means - hull.mean(0)) <=
 * 0.2 * scale_factor``, dn_model.py:1255-1257); the others keep ~0. */
int fsgs_nearest_point_words(int nq, const float *queries, int np, const float *points, const float *center,
                             float close_radius, uint64_t *out_words, fsgs_stream_t stream);
/* The k nearest points (exact fp32 differences, brute force, ties -> lowest index) of every query, reported from rank
 * `skip` on: out_idx [nq, k - skip] int64.  k <= 33, k <= np; skip = 1 reproduces dn_splatter/utils/knn.py:29-44
 * (knn_sk asks sklearn for k + 1 neighbours and drops the first column) — what compute_level_surface_points
 * (dn_model.py:1762-1764) tracks per back-projected pixel.  No counterpart in gsplat. */
int fsgs_knn_points(int64_t nq, const float *queries, int np, const float *points, int k, int skip, int64_t *out_idx,
                    fsgs_stream_t stream);
/* split_gaussians sample kernel: for every selected parent p (ids[S]) and sample s<n_samples,
 * new_mean = mean[p] + R(q[p]/|q|) (exp(log_scale[p]) * z[s*S+i]); new_log_scale = log(exp(ls)/1.6).
 * Writes new_means[n_samples*S,3], new_log_scales[n_samples*S,3] (sample-major, like .repeat). */
int fsgs_split_samples(int64_t S, int n_samples, const int64_t *ids, const float *means,
                       const float *quats, const float *log_scales, const float *randn,
                       float *new_means, float *new_log_scales, fsgs_stream_t stream);

/* ---- a-13 / a-14 in two launches (ABI 10): mark -> [the host reads five totals] -> move ---------------------------------
 * One refinement of dn_splatter/dn_model.py:326-451 (split / duplicate selection :342-379, split_gaussians' children,
 * cull_gaussians :403-431) or one cull of the pruning callbacks (:1156-1302), with the Adam-state surgery of
 * dup_in_all_optim / remove_from_all_optim (:1120-1152), as the one-pass kernel SURVEY.md section 7 step 7 asks for.
 * Rounds 1-5 ran the masks, torch.where / cat / repeat and per-tensor compactions as ~80 torch launches per refinement.
 *
 * fsgs_refine_mark decides, per existing row, five bits of flags[row]:
 *   1 KEEP        the row survives (not low-alpha, not too big, not a split parent, none of the pruning tests below)
 *   2 SPLIT       densify only: (exp(scale).max > densify_size_thresh | check_screen & max_2Dsize > split_screen_size)
 *                 & avg_grad_norm > densify_grad_thresh & !add_mask, avg_grad_norm = xys_grad_norm / vis_counts * 0.5 * max_hw
 *   4 DUP         densify only: scale max AFTER the split's /1.6 <= densify_size_thresh & high gradient & !add_mask (the
 *                 reference tests the duplicates after split_gaussians has shrunk the parents in place: a parent just above
 *                 the threshold is both split and duplicated)
 *   8 CHILD_KEEP  the row's split children pass cull_gaussians (the parent's opacity, the shrunk scales)
 *  16 DUP_KEEP    its duplicate passes it
 * and leaves, in book (int32 [fsgs_refine_book_ints(N)], ZERO before the first call, self-resetting), the exclusive
 * per-workgroup (256 rows) offsets of the five counts {KEEP, SPLIT, DUP, SPLIT & CHILD_KEEP, DUP & DUP_KEEP}; the five
 * totals go to totals_mapped[0..4] (mapped host memory), then totals_mapped[7] <- 1 with system-scope release.
 * Pruning tests riding in the same pass (hull_pruning / touch_pruning, :1249-1302): hull_best (nullable) = the 64-bit
 * words fsgs_nearest_point left for means against the visual hull (distance bits above index bits, ~0 = none):
 * culled when |mean - hull_center| <= hull_close and hull_lo < distance <= hull_hi; or, without a search launch at all,
 * hull_points (float4 per hull point, sorted by cell) + hull_cells (int32 [cells + 1], first point of every cell) of a
 * uniform grid over the hull whose cell edge exceeds hull_hi: the mark then looks for the nearest hull point in the 27
 * cells around a close row — the decision is the exhaustive search's, because a row whose nearest hull point is not
 * in those cells is farther than hull_hi from all of them (fusionsense_amd/touch.py: hull_grid); boxes (nullable, n_boxes x 18 floats as
 * for fsgs_points_in_boxes): culled when inside any.  Rows of add_mask (touch anchors) pass both.  extra_cull (nullable):
 * a byte per row, non-zero = culled (the caller's own test).
 * xys_grad_norm / vis_counts are read only when rules->densify; max_2Dsize is nullable (no screen-size tests then). */
typedef struct fsgs_refine_rules {
    int32_t densify;              /* 1: split / dup selection + cull; 0: cull only */
    int32_t n_samples;            /* children per split parent (SplatfactoModelConfig.n_split_samples) */
    float max_hw;                 /* max(H, W) of the last training frame */
    float densify_grad_thresh, densify_size_thresh;
    int32_t check_screen;         /* step < stop_screen_size_at */
    float split_screen_size;
    float cull_alpha_thresh;
    int32_t check_big;            /* step > refine_every * reset_alpha_every */
    float cull_scale_thresh, cull_screen_size;
    float hull_center[3];
    float hull_close, hull_lo, hull_hi;
    int32_t n_boxes;
    float grid_origin[3];         /* hull_cells route: cell (x, y, z) of a point p = floor((p - grid_origin) * grid_inv_cell) */
    float grid_inv_cell;          /* 1 / cell edge, the edge > hull_hi */
    int32_t grid_dims[3];         /* cells per axis (x fastest): cell id = (z * dims[1] + y) * dims[0] + x */
} fsgs_refine_rules;
int64_t fsgs_refine_book_ints(int64_t N);
int fsgs_refine_mark(int64_t N, const fsgs_refine_rules *rules, const float *xys_grad_norm, const float *vis_counts,
                     const float *max_2Dsize, const float *means, const float *log_scales, const float *opac_logit,
                     const uint8_t *add_mask, const uint8_t *extra_cull, const uint64_t *hull_best, const float *hull_points,
                     const int32_t *hull_cells, const float *boxes, uint8_t *flags, int32_t *book, int32_t *totals_mapped,
                     fsgs_stream_t stream);
/* fsgs_refine_move builds the new tensors from flags / book and the totals the host has read: for each of n_cols <= 24
 * columns (row-major fp32 [N, row_floats[c]]) dst[c] receives, in the reference's order,
 *   [kept old rows] [for s < n_samples: the kept children of sample s, parents in row order] [kept duplicates] [n_append rows]
 * A column's kind says what a NEW row holds: 0 COPY = the parent's row (append rows: append[c]), 1 ZERO (Adam moments of
 * new rows, dup_in_optim), 2 MEANS = child: mean + R(q/|q|) (exp(log_scale) * randn[s * n_split + i]) with i the parent's
 * rank among ALL split rows (kept or not), 3 SCALES = child: log(exp(scale) / 1.6); duplicate of a split parent: the same.
 * quats / log_scales / randn [n_samples * n_split, 3] are read for kind 2 only (nullable without splits).
 * mask_in -> mask_out (nullable): a byte column (add_mask): kept old rows keep theirs, children / duplicates get 0, append rows
 * mask_append.  append[c] nullable when n_append == 0 or kind 1.  dst rows: n_keep + n_samples * n_split_kept + n_dup_kept + n_append. */
int fsgs_refine_move(int64_t N, int n_cols, const float *const *src, float *const *dst, const float *const *append,
                     const int *row_floats, const int *kind, const uint8_t *flags, const int32_t *book,
                     int64_t n_keep, int64_t n_split, int64_t n_split_kept, int64_t n_dup_kept, int64_t n_append, int n_samples,
                     const float *randn, const float *quats, const float *log_scales,
                     const uint8_t *mask_in, uint8_t *mask_out, int mask_append, fsgs_stream_t stream);

/* ---- caller-side glue of get_outputs, fused (csrc/glue.hip; used by fusionsense_amd/fused.py) -----
 * activations of dn_model.py:573-574 and their VJPs (v_quats = v_quats_a + v_quats_b sums the
 * projection and normal-pass gradient streams; v_quats_b nullable). */
int fsgs_activate_fwd(int N, const float *log_scales, const float *opac_logit, float *scales,
                      float *opac, fsgs_stream_t stream);
int fsgs_activate_bwd(int N, const float *scales, const float *opac, const float *v_scales,
                      const float *v_opac, const float *v_quats_a, const float *v_quats_b,
                      float *v_log_scales, float *v_opac_logit, float *v_quats, fsgs_stream_t stream);
/* fsgs_project_fwd with the activations of dn_model.py:573-574 applied in the same launch:
 * scales_out [N,3] = exp(log_scales), opac_out [N] = sigmoid(opac_logit); the projection uses scales_out.
 * binarise != 0: first opac_logit[n] = opac_logit[n] >= binary_threshold ? 1 : 0, written back to the parameter
 * (the binary-opacity write at the top of get_outputs, dn_model.py:492-503). */
int fsgs_project_fwd_act(int C, int N, const float *means, const float *quats, const float *log_scales,
                         float *opac_logit, int binarise, float binary_threshold,
                         const float *viewmats, const float *Ks, int width,
                         int height, float eps2d, float near_plane, float far_plane, float radius_clip,
                         float *scales_out, float *opac_out, int32_t *radii, float *means2d, float *depths,
                         float *conics, fsgs_stream_t stream);
/* The per-Gaussian tail of the fused backward in ONE launch (C == 1): reads each Gaussian's packed
 * gradient record (fsgs_raster_bwd_quad; cleared afterwards), applies the VJP of the projection
 * (as fsgs_project_bwd with v_means2d / v_conics / v_depths taken from the record), of the normal pass
 * (fsgs_normals_bwd), of exp(scales) / sigmoid(opacities) (fsgs_activate_bwd), writes absgrad [N,2] and,
 * when the three statistics arrays are given, applies fsgs_densify_stats.  scales = exp(log_scales),
 * opac = sigmoid(opacity logits); accumulate_means != 0: v_means += (after fsgs_sh_bwd_split wrote it). */
int fsgs_gaussian_bwd(int N, const float *means, const float *quats, const float *log_scales,
                      const float *scales, const float *opac, const float *viewmat, const float *K,
                      const float *c2w, int width, int height, float eps2d, const int32_t *radii,
                      const float *conics, float *v_packed, int accumulate_means, float *v_means,
                      float *v_quats, float *v_log_scales, float *v_opac_logit, float *absgrad,
                      float *xys_grad_norm, float *vis_counts, float *max_2Dsize, float inv_max_hw,
                      const uint8_t *frozen, int64_t replica_rows,
                          fsgs_stream_t stream);
/* flags of fsgs_gauss_sh_bwd / _h16 / _adam / _adam_h16 (per launch; the outputs are the same numbers either way):
 *   FSGS_GSB_LAZY_COEFFS  a Gaussian's SH coefficients are fetched only after its gradient line, and only if the line
 *                         carries a colour gradient (dense scenes: most lines are empty; 192 B less read per empty line,
 *                         at the price of a dependent load);
 *   FSGS_GSB_SKIP_IDLE    (_adam) an element with zero gradient on zero moments is left alone: its moments are read
 *                         first and the parameter only if something changes (8 instead of 24 B for such a float, a
 *                         dependent load for the others) — for scenes most of whose Gaussians no view has reached yet;
 *                         without it parameter and moments are read together and every element is stepped.
 * DEPRECATED: flags < 0 = both on from the process-wide threshold of fsgs_set_lazy_sh_min_n on (default 2^20, env
 * FSGS_LAZY_SH_MIN_N; returns the previous value), the round-3 behaviour. */
#define FSGS_GSB_LAZY_COEFFS 1
#define FSGS_GSB_SKIP_IDLE 2
int fsgs_set_lazy_sh_min_n(int n);

/* fsgs_sh_bwd_split (or, with v_rgb_masked != NULL, fsgs_sh_bwd_colors) for one camera, K = 16 stored coefficients
 * and the packed 16-float gradient records, followed by fsgs_gaussian_bwd — in ONE launch and one thread per
 * Gaussian: the record is read (replicas folded, everything cleared) once and the view-direction share of v_means
 * never leaves the registers.  Same results as the two calls (which stay for K != 16, several cameras and half
 * storage).  Replaces the same reference calls as they do. */
int fsgs_gauss_sh_bwd(int N, int degree, const float *means, const float *campos, const float *features_dc,
                      const float *features_rest, const float *quats, const float *log_scales, const float *scales,
                      const float *opac, const float *viewmat, const float *K, const float *c2w, int width, int height,
                      float eps2d, const int32_t *radii, const float *conics, float *v_packed, float *v_features_dc,
                      float *v_features_rest, float *v_rgb_masked, float *v_means, float *v_quats, float *v_log_scales,
                      float *v_opac_logit, float *absgrad, float *xys_grad_norm, float *vis_counts, float *max_2Dsize,
                      float inv_max_hw, const uint8_t *frozen, int64_t replica_rows, int flags, fsgs_stream_t stream);
/* fsgs_gauss_sh_bwd on half attribute storage (features, quats, log_scales read from IEEE-half mirrors; all
 * gradients fp32; no factored output). */
int fsgs_gauss_sh_bwd_h16(int N, int degree, const float *means, const float *campos, const void *features_dc_h,
                          const void *features_rest_h, const void *quats_h, const void *log_scales_h,
                          const float *scales, const float *opac, const float *viewmat, const float *K, const float *c2w,
                          int width, int height, float eps2d, const int32_t *radii, const float *conics, float *v_packed,
                          float *v_features_dc, float *v_features_rest, float *v_means, float *v_quats,
                          float *v_log_scales, float *v_opac_logit, float *absgrad, float *xys_grad_norm,
                          float *vis_counts, float *max_2Dsize, float inv_max_hw, const uint8_t *frozen,
                          int64_t replica_rows, int flags, fsgs_stream_t stream);
/* fsgs_gauss_sh_bwd / _h16 with the Adam step of all six parameter groups (dn_config.py:36-75) applied where the
 * gradients are formed: no gradient is written (236 B per Gaussian less written here and less read by the Adam launch
 * this replaces; same update, bit for bit, as fsgs_adam_step on the gradients fsgs_gauss_sh_bwd writes).  adam: exactly
 * six groups in the order means [N,3], log-scales [N,3], quats [N,4], features_dc [N,3], features_rest [N,45], opacity
 * logits [N,1]; grads[] is ignored; half_mirror[] entries (nullable; required for all but the means by _h16) are
 * rewritten with the update.  A Gaussian's parameters move after the thread that owns it has read them; nothing else in
 * the launch reads them.  min_scale_g != 0: the gradient of get_loss_dict's two_d_gaussians term (dn_model.py:817-819;
 * what fsgs_min_scale_loss(v_loss = 1, g = min_scale_g) adds to the log-scale gradients after the backward) is added to
 * the log-scale gradients here, from the fp32 masters.  For single-rank steps whose gradients nobody else needs. */
int fsgs_gauss_sh_bwd_adam(int N, int degree, const float *means, const float *campos, const float *features_dc,
                           const float *features_rest, const float *quats, const float *log_scales, const float *scales,
                           const float *opac, const float *viewmat, const float *K, const float *c2w, int width,
                           int height, float eps2d, const int32_t *radii, const float *conics, float *v_packed,
                           float *absgrad, float *xys_grad_norm, float *vis_counts, float *max_2Dsize, float inv_max_hw,
                           const uint8_t *frozen, int64_t replica_rows, const fsgs_adam_groups *adam, float min_scale_g,
                           int flags, fsgs_stream_t stream);
int fsgs_gauss_sh_bwd_adam_h16(int N, int degree, const float *means, const float *campos, const void *features_dc_h,
                               const void *features_rest_h, const void *quats_h, const void *log_scales_h,
                               const float *scales, const float *opac, const float *viewmat, const float *K,
                               const float *c2w, int width, int height, float eps2d, const int32_t *radii,
                               const float *conics, float *v_packed, float *absgrad, float *xys_grad_norm,
                               float *vis_counts, float *max_2Dsize, float inv_max_hw, const uint8_t *frozen,
                               int64_t replica_rows, const fsgs_adam_groups *adam, float min_scale_g,
                               int flags, fsgs_stream_t stream);
/* frozen (nullable, [N] u8): rows whose v_means / v_log_scales / v_opac_logit are zero — FusionSense's touch
 * anchors, detached at dn_model.py:535-541 (their quaternion and colour gradients still flow). */
/* dn_model.py:602-613, 655-656: rgb = clamp(render[:3] + (1-alpha) bg, 0, 1); depth = alpha > 0 ?
 * render[3] : max(render[3]); normal = (n/|n| + 1)/2.  render [P,4], alphas [P], render_extra [P,3],
 * bg [3]; n_partial > 0: max_last_partial [n_partial] (per-workgroup partial maxima) is reduced into max_last[0]
 * first; n_partial <= 0: max_last already holds max(1, -n_partial) partial maxima.  bwd: any of v_rgb / v_depth / v_normal /
 * v_alpha_in may be NULL (= zero); writes v_render [P,4], v_alphas [P], v_render_extra [P,3].
 * ALIGNMENT: the forward epilogues (fsgs_epilogue_fwd, _loss_fwd, _fwd_order) move four pixels per lane with 16-byte
 * accesses: render, alphas, render_extra, rgb, depth, normal, depth_gt, normal_gt, v_depth, v_normal must be 16-byte
 * aligned (any allocation's start is; a view at an odd pixel offset is not) — FSGS_EINVAL otherwise. */
int fsgs_epilogue_fwd(int64_t n_pixels, const float *render, const float *alphas,
                      const float *render_extra, const float *bg, const float *max_last_partial,
                      int n_partial, float *max_last, float *rgb, float *depth, float *normal,
                      fsgs_stream_t stream);
/* fsgs_epilogue_fwd (max_last = n_cells partial image maxima, as fsgs_raster_fwd_quad leaves them) and
 * fsgs_aux_l1_fwd_bwd in one pass over the pixels, for a caller that knows the targets and the upstream gradient of
 * the loss when the images are formed: partial [ceil(n_pixels / 256), 2], v_depth, v_normal as there. */
int fsgs_epilogue_loss_fwd(int64_t n_pixels, const float *render, const float *alphas, const float *render_extra,
                           const float *bg, const float *max_last, int n_cells, float *rgb, float *depth,
                           float *normal, const float *depth_gt, const float *normal_gt, const float *v_loss,
                           float g_depth, float g_normal, float *partial, float *v_depth, float *v_normal,
                           fsgs_stream_t stream);
/* fsgs_epilogue_loss_fwd (depth_gt != NULL) or fsgs_epilogue_fwd over the forward's n_cells partial maxima (depth_gt ==
 * NULL: no loss terms; v_loss / partial / v_depth / v_normal unused) — and, riding in the launch as extra workgroups, the
 * dispatch order of the compositing backward: bwd_order != NULL -> the counting sort described at fsgs_raster_fwd_quad
 * (n_rec, seg_split [4, th * tw] as the forward left them; order_counters = the 32 zeroed words behind bwd_queue's items). */
int fsgs_epilogue_fwd_order(int64_t n_pixels, const float *render, const float *alphas, const float *render_extra,
                            const float *bg, const float *max_last, int n_cells, float *rgb, float *depth, float *normal,
                            const float *depth_gt, const float *normal_gt, const float *v_loss, float g_depth,
                            float g_normal, float *partial, float *v_depth, float *v_normal, const int32_t *n_rec,
                            const int32_t *seg_split, int32_t *order_counters, int32_t *bwd_order,
                            int order_shift /* class = min(own records >> order_shift, 31) */, int tile_width,
                            int tile_height, fsgs_stream_t stream);
int fsgs_epilogue_bwd(int64_t n_pixels, const float *render, const float *alphas,
                      const float *render_extra, const float *bg, const float *v_rgb,
                      const float *v_depth, const float *v_normal, const float *v_alpha_in,
                      float *v_render, float *v_alphas, float *v_render_extra, fsgs_stream_t stream);

/* ---- N1: torch.optim.Adam (amsgrad=False, weight_decay=0) for up to 8 parameter groups in one
 * launch (dn_splatter/dn_config.py:36-75 steps one optimizer per group).  Arrays of n_groups HOST
 * entries holding device pointers; step is the 1-based step count after the increment. */
int fsgs_adam_step(int n_groups, float *const *params, const float *const *grads, float *const *exp_avg,
                   float *const *exp_avg_sq, const int64_t *numel, const float *lr, int step, double beta1,
                   double beta2, float eps, fsgs_stream_t stream);

/* ---- BASELINE config #5: half-precision attribute storage ----------------------------------------------------
 * The render path can read the per-Gaussian attributes other than the means — SH features, log-scales, quaternions,
 * opacity logits — from IEEE-half MIRRORS of the fp32 master parameters: 124 instead of 236 parameter bytes per
 * Gaussian per frame.  All arithmetic and every gradient stay fp32; Adam updates the masters and rewrites the
 * mirrors in the same launch.  The *_h16 entries take the mirrors (const void * = half) where their fp32 twins
 * take floats and are otherwise identical, argument for argument:
 *   fsgs_project_bin_live_count_h16 / fsgs_project_fwd_act_h16   (+ opac_logit_master, nullable: the binary-opacity
 *       write goes to mirror and master), fsgs_sh_fwd_pack_h16, fsgs_sh_bwd_split_h16 (one camera),
 *   fsgs_gaussian_bwd_h16, fsgs_adam_step_h16 (half_mirrors[n_groups], nullable entries). */
int fsgs_project_bin_live_count_h16(int N, const float *means, const void *quats_h, const void *log_scales_h,
                                    void *opac_logit_h, float *opac_logit_master, int binarise, float binary_threshold,
                                    const float *viewmat, const float *K, int width, int height, float eps2d,
                                    float near_plane, float far_plane, float radius_clip, float *scales_out,
                                    float *opac_out, int32_t *radii, float *means2d, float *depths, float *conics,
                                    int tile_width, int tile_height, int32_t *tiles_per_gauss, int32_t *isect_offsets,
                                    void *table_scratch, size_t table_bytes, int32_t *n_live_mapped,
                                    fsgs_stream_t stream);
int fsgs_project_fwd_act_h16(int C, int N, const float *means, const void *quats_h, const void *log_scales_h,
                             void *opac_logit_h, float *opac_logit_master, int binarise, float binary_threshold,
                             const float *viewmats, const float *Ks, int width, int height, float eps2d,
                             float near_plane, float far_plane, float radius_clip, float *scales_out, float *opac_out,
                             int32_t *radii, float *means2d, float *depths, float *conics, fsgs_stream_t stream);
int fsgs_sh_fwd_pack_h16(int N, int K, int degree, const float *means, const float *campos, const void *features_dc_h,
                         const void *features_rest_h, const int32_t *radii, const float *depths, const float *means2d,
                         const float *conics, const float *opacities, const void *quats_h, const void *log_scales_h,
                         const float *c2w, float *packed, float *normals_world, float *zero_cells, int n_zero,
                         fsgs_stream_t stream);
int fsgs_sh_bwd_split_h16(int N, int K, int degree, const float *means, const float *campos, const void *features_dc_h,
                          const void *features_rest_h, const int32_t *radii, int D, const float *v_colors,
                          float *v_features_dc, float *v_features_rest, float *v_means, float *v_depths,
                          int overwrite_means, int64_t replica_rows, fsgs_stream_t stream);
int fsgs_gaussian_bwd_h16(int N, const float *means, const void *quats_h, const void *log_scales_h, const float *scales,
                          const float *opac, const float *viewmat, const float *K, const float *c2w, int width,
                          int height, float eps2d, const int32_t *radii, const float *conics, float *v_packed,
                          int accumulate_means, float *v_means, float *v_quats, float *v_log_scales,
                          float *v_opac_logit, float *absgrad, float *xys_grad_norm, float *vis_counts,
                          float *max_2Dsize, float inv_max_hw, const uint8_t *frozen, int64_t replica_rows,
                          fsgs_stream_t stream);
int fsgs_adam_step_h16(int n_groups, float *const *params, const float *const *grads, float *const *exp_avg,
                       float *const *exp_avg_sq, void *const *half_mirrors, const int64_t *numel, const float *lr,
                       int step, double beta1, double beta2, float eps, fsgs_stream_t stream);

/* ---- N2: photometric loss on the render, fused (dn_splatter/dn_model.py:683 main loss with the
 * torchmetrics SSIM(kernel_size=11) of :244).  pred, gt: [H,W,3] channel-last.
 * fwd: sums[P,2] per-workgroup partials (P = fsgs_ssim_l1_num_partials(H,W)): column 0 sums to
 * sum |pred-gt|, column 1 to the sum of the SSIM map over the (H-10)x(W-10) interior; plus the
 * three partial-derivative maps (planar [3,H,W]) the backward needs.
 * bwd: v_pred = v_loss[0] * (g_l1 * sign(pred-gt) + g_ssim * dSSIMsum/dpred). */
int64_t fsgs_ssim_l1_num_partials(int H, int W);
int fsgs_ssim_l1_fwd(int H, int W, const float *pred, const float *gt, float *dm_dmu1,
                     float *dm_dsigma1, float *dm_dsigma12, float *sums, fsgs_stream_t stream);
int fsgs_ssim_l1_bwd(int H, int W, const float *pred, const float *gt, const float *dm_dmu1,
                     const float *dm_dsigma1, const float *dm_dsigma12, const float *v_loss,
                     float g_l1, float g_ssim, float *v_pred, fsgs_stream_t stream);
/* fsgs_ssim_l1_bwd and fsgs_loss_combine in one launch (arguments of both). */
int fsgs_ssim_l1_bwd_combine(int H, int W, const float *pred, const float *gt, const float *dm_dmu1,
                             const float *dm_dsigma1, const float *dm_dsigma12, const float *v_loss, float g_l1,
                             float g_ssim, float *v_pred, int n_terms, const float *const *partials,
                             const int64_t *rows, const float *weights, float bias, float *loss_out,
                             fsgs_stream_t stream);

/* Auxiliary L1 terms on the depth [P] and normal [P,3] images (normal nullable), fused:
 * fwd: partial[ceil(P/256), 2] per-workgroup sums of |depth-gt| and |normal-gt|;
 * bwd: v_depth = v_loss[0]*g_depth*sign(depth-gt), v_normal likewise (written). */
int fsgs_aux_l1_fwd(int64_t n_pixels, const float *depth, const float *depth_gt, const float *normal,
                    const float *normal_gt, float *partial, fsgs_stream_t stream);
int fsgs_aux_l1_bwd(int64_t n_pixels, const float *depth, const float *depth_gt, const float *normal,
                    const float *normal_gt, const float *v_loss, float g_depth, float g_normal,
                    float *v_depth, float *v_normal, fsgs_stream_t stream);
/* fsgs_aux_l1_fwd and fsgs_aux_l1_bwd in one pass, for callers that know the upstream gradient of the loss
 * when they evaluate it (v_loss[0], device): partial sums as fsgs_aux_l1_fwd, gradient images as fsgs_aux_l1_bwd. */
int fsgs_aux_l1_fwd_bwd(int64_t n_pixels, const float *depth, const float *depth_gt, const float *normal,
                        const float *normal_gt, float *partial, const float *v_loss, float g_depth,
                        float g_normal, float *v_depth, float *v_normal, fsgs_stream_t stream);

/* The scalar loss from the partials above without torch reductions or a host sync:
 * out[0] = bias + sum_t (weights[2t] * sum_r partials[t][r,0] + weights[2t+1] * sum_r partials[t][r,1]),
 * t < n_terms <= 6; partials[t] is [rows[t],2] on the device, the three arrays are HOST arrays.
 * (dn_model.py:673-925 adds its terms with python scalars; the sum is accumulated in f64.) */
int fsgs_loss_combine(int n_terms, const float *const *partials, const int64_t *rows,
                      const float *weights, float bias, float *out, fsgs_stream_t stream);
/* General form: partials[t] is [rows[t], cols[t]] (cols[t] <= 8, n_terms <= 6); weights holds cols[t] consecutive
 * floats per term, one per column.  cols == NULL: two columns per term (fsgs_loss_combine). */
int fsgs_loss_combine_cols(int n_terms, const float *const *partials, const int64_t *rows, const int *cols,
                           const float *weights, float bias, float *out, fsgs_stream_t stream);

/* ---- a-15: the FusionSense training loss, DNSplatterModel.get_loss_dict (dn_splatter/dn_model.py:673-925) ----
 * Photometric term with the object mask (splatfacto get_loss_dict called at dn_model.py:683 multiplies both
 * images by batch["mask"]): mask [H,W] float or NULL; pred and gt are multiplied by it as they are loaded and
 * v_pred = mask * d loss / d(pred * mask).  The backward optionally carries the combine of all loss partials
 * (loss_out != NULL; arguments of fsgs_loss_combine_cols). */
int fsgs_ssim_l1_fwd_masked(int H, int W, const float *pred, const float *gt, const float *mask, float *dm_dmu1,
                            float *dm_dsigma1, float *dm_dsigma12, float *sums, fsgs_stream_t stream);
int fsgs_ssim_l1_bwd_masked(int H, int W, const float *pred, const float *gt, const float *mask,
                            const float *dm_dmu1, const float *dm_dsigma1, const float *dm_dsigma12,
                            const float *v_loss, float g_l1, float g_ssim, float *v_pred, int n_terms,
                            const float *const *partials, const int64_t *rows, const int *cols,
                            const float *weights, float bias, float *loss_out, fsgs_stream_t stream);

/* Depth and normal terms of get_loss_dict in ONE pass over the images (dn_model.py:702-764, 770-815;
 * dn_splatter/losses.py:177-214 EdgeAwareLogL1, :269-285 TVLoss), with d = depth*mask, g = sensor*mask,
 * n = normal*mask, n* = normal_gt*mask, valid = g > depth_tol, I = clamp(image, min 10/255):
 *   col 0  sum over valid, x < W-1 of exp(-mean_c|I(x)-I(x+1)|) * log(1+|d-g|)      (EdgeAwareLogL1, x)
 *   col 1  the same along y                                                            (EdgeAwareLogL1, y)
 *   col 2  sum_{x<W-1} |d(x)-d(x+1)|        col 3  sum_{y<H-1} |d(y)-d(y+1)|           (TV on depth)
 *   col 4  sum |n-n*| over 3 channels                                                  (normal L1)
 *   col 5  sum_{x<W-1} |n(x)-n(x+1)|        col 6  sum_{y<H-1} |n(y)-n(y+1)|           (TV on normals)
 *   col 7  number of valid pixels with x < W-1 ... unused (0)
 * partial: [fsgs_fusion_aux_num_partials(H,W), 8] per-workgroup sums.  w[7]: the weight of every column in the
 * loss (lambda / count; the two EdgeAwareLogL1 counts are per-view constants, fsgs_depth_valid_counts).
 * v_loss != NULL: also writes v_depth [H,W] and v_normal [H,W,3] = v_loss[0] * d loss / d image (mask applied).
 * normal / normal_gt / mask nullable (columns 4-6 then 0).
 * flags (round 4: the switches of get_loss_dict that FusionSense's configuration leaves off, 0 = none):
 *   FSGS_FA_NORMAL_GT_UNMASKED  n* = normal_gt as given (the pseudo normals of fsgs_normals_from_depth, which
 *                               dn_model.py:774-795 does not multiply by the mask), not normal_gt * mask;
 *   FSGS_FA_EDGE_AWARE_TV       cols 2 / 3 = EdgeAwareTV (losses.py:241-266): |d(x)-d(x+1)| * exp(-mean_c|I(x)-I(x+1)|);
 *   FSGS_FA_DEPTH_L1 / _LOGL1 / _MSE  the plain depth-loss types of dn_model.py:731-736 (losses.py:147-174,
 *                               torch.nn.MSELoss) over the valid pixels: col 0 = sum |d-g| / log(1+|d-g|) / (d-g)^2,
 *                               col 1 = 0; w[0] = lambda / #valid (counts[2] of fsgs_depth_valid_counts). */
#define FSGS_FA_NORMAL_GT_UNMASKED 1
#define FSGS_FA_EDGE_AWARE_TV 2
#define FSGS_FA_DEPTH_L1 4
#define FSGS_FA_DEPTH_LOGL1 8
#define FSGS_FA_DEPTH_MSE 12
int64_t fsgs_fusion_aux_num_partials(int H, int W);
int fsgs_fusion_aux_loss(int H, int W, const float *depth, const float *normal, const float *image,
                         const float *sensor_depth, const float *normal_gt, const float *mask, float depth_tol,
                         const float *w, const float *v_loss, float *partial, float *v_depth, float *v_normal,
                         int flags, fsgs_stream_t stream);
/* fsgs_fusion_aux_loss with the partial sums of fsgs_min_scale_loss (forward only: g = 0, no gradient) and
 * fsgs_touch_normal_sqerr riding in the same launch as extra workgroups: N > 0 -> min_scale_partial [ceil(N / 256), 2],
 * n_touch > 0 -> touch_partial [ceil(n_touch / 256), 2], the same values as the stand-alone calls (two launches less on
 * FusionSense's training step). */
int fsgs_fusion_aux_loss_riders(int H, int W, const float *depth, const float *normal, const float *image,
                                const float *sensor_depth, const float *normal_gt, const float *mask, float depth_tol,
                                const float *w, const float *v_loss, float *partial, float *v_depth, float *v_normal,
                                int flags, int N, const float *log_scales, float *min_scale_partial, int n_touch,
                                const int64_t *touch_idx, const float *normals_world, const float *touch_normals,
                                float *touch_partial, fsgs_stream_t stream);
/* get_loss_dict's normal_supervision == "depth" target (dn_model.py:774-795; utils/normal_utils.py:8-46 over
 * utils/camera_utils.py:92-144 with an identity pose): pseudo normals of depth * mask — interior pixels
 * normalize(cross(right - left, top - bottom)) of the back-projected pixel centres, border zero — with y and z negated,
 * mapped to [0,1]: normal_out [H,W,3] = (1 + n * (1,-1,-1)) / 2.  (fx, fy, cx, cy): the camera of the frame. */
int fsgs_normals_from_depth(int H, int W, const float *depth, const float *mask, float fx, float fy, float cx, float cy,
                            float *normal_out, fsgs_stream_t stream);
/* use_normal_cosine_loss (dn_model.py:807-813) AS CALLED there: metrics.mean_angular_error (metrics.py:58-73) on
 * [3,H,W] tensors sums over the image rows, so the term is mean over (channel, column) of
 * acos(clamp(sum_y ((n*-1)/2)((n-1)/2), -1, 1)), n = normal * mask, n* = normal_gt (* mask unless gt_unmasked).
 * partial [fsgs_normal_cosine_num_partials(W), 2]: col 0 = sum of the acos values (weight normal_lambda / (3 W));
 * v_loss != NULL: v_normal [H,W,3] += v_loss[0] * w * d/d normal (ACCUMULATED onto fsgs_fusion_aux_loss's output). */
int64_t fsgs_normal_cosine_num_partials(int W);
int fsgs_normal_cosine_loss(int H, int W, const float *normal, const float *normal_gt, const float *mask,
                            int gt_unmasked, float w, const float *v_loss, float *partial, float *v_normal,
                            fsgs_stream_t stream);
/* counts[0] = #{valid, x < W-1}, counts[1] = #{valid, y < H-1}, counts[2] = #{valid} with valid = sensor*mask > depth_tol
 * (the sizes of the two masked selections of losses.py:208-209 and of the plain selection of dn_model.py:733);
 * device int64[3], zeroed by the call. */
int fsgs_depth_valid_counts(int H, int W, const float *sensor_depth, const float *mask, float depth_tol,
                            int64_t *counts, fsgs_stream_t stream);
/* two_d_gaussians term (dn_model.py:817-819): partial[ceil(N/256), 2] col 0 = sum_n min_k exp(log_scales[n,k]);
 * v_loss != NULL: g_log_scales[n, argmin] += v_loss[0] * g * exp(min) (accumulated: runs after the rasterizer's
 * own gradient has been written; first minimum on ties). */
int fsgs_min_scale_loss(int N, const float *log_scales, float g, const float *v_loss, float *partial,
                        float *g_log_scales, fsgs_stream_t stream);
/* touch-normal MSE (dn_model.py:893-902): partial[ceil(n/256), 2] col 0 = sum over the n anchor rows idx[i] of
 * |normals_world[idx[i]] - touch_normals[i]|^2.  Value only: the reference's normals entry is a detached leaf. */
int fsgs_touch_normal_sqerr(int n, const int64_t *idx, const float *normals_world, const float *touch_normals,
                            float *partial, fsgs_stream_t stream);

/* ---- One training step as ONE call (round 6).  `DNSplatterModel.get_outputs` (dn_model.py:469-671: rasterization() at
 * :570-591 + the legacy normal pass at :644-653 + the image epilogue :602-613, 655-664), the loss on its images, both
 * backward passes, nerfstudio's after_train statistics (registered at dn_model.py:1385-1389) and the Adam step of the six
 * Gaussian parameter groups (dn_config.py:36-75) — the launches the per-op entry points above enqueue one by one when a
 * host drives them (fusionsense_amd/fused.py), here enqueued back to back by the library from ONE argument block, so that
 * issuing a step costs the host microseconds instead of ~0.45 ms of interpreter time.  Nothing new runs on the device:
 * every launch is one of the entry points above with the arguments named here; results are theirs, bit for bit.
 *
 * The route is the COUNT-FREE one (fsgs_project_bin_live_fill_sh_pack): one camera, fp32 attributes, 16 stored SH
 * coefficients, degree <= 3, no occlusion cuts, a view whose previous frame left bucket room (`bucket_base`).  Loss: the
 * benchmark loss of BASELINE config #2 ((1 - l) L1 + l (1 - SSIM11) on rgb, plain L1 on depth / normal).
 * Frames that do not qualify (first visit of a view, half storage, dense scenes, get_loss_dict's terms, several ranks)
 * keep the per-op route; so does the frame that is redone after an overflow.
 *
 *   fsgs_step_forward   launches 1-5: project + bin + SH / pack | in-tile sorts | compositing forward | image epilogue
 *                       with the depth / normal L1 terms and the backward's dispatch order | SSIM forward
 *   fsgs_step_backward  waits (bounded spin on the mapped flag the binning's bookkeeping workgroup raises, then a stream
 *                       synchronise) for the frame's live total, returns FSGS_STEP_OVERFLOW (> 0) WITHOUT launching
 *                       anything if the lists were truncated (total > capacity) or a tile outgrew its bucket — nothing
 *                       with side effects has run by then: statistics, gradient accumulator, parameters and moments are
 *                       untouched and the caller redoes the frame through the exact two-pass route — else launches 6-8:
 *                       SSIM backward + loss combine | compositing backward | per-Gaussian backward + statistics + Adam
 *   fsgs_step_run       both, back to back
 * n_live_out (nullable): the frame's true number of live pairs (valid after fsgs_step_backward / _run, also on overflow).
 *
 * The block is PLAIN DATA owned by the caller; the library keeps no copy and no state.  Every pointer is device memory
 * unless marked (host) / (mapped).  `mapped` = int32[4] in host memory the device can write (hipHostMalloc mapped /
 * a pinned torch tensor): [0] live total, [1] done flag, [2] capacity (written by fsgs_step_forward), [3] bucket
 * overflow; fsgs_step_forward clears [1] and [3]; a block must not be passed to fsgs_step_forward again before
 * fsgs_step_backward (or _run) has returned for it — FSGS_EPROTOCOL otherwise (`armed`, the one field the calls write).
 * Buffers marked [frame] are outputs a caller may read after the step; [scratch] are overwritten by every step. */
#define FSGS_STEP_OVERFLOW 1
typedef struct fsgs_step_plan {
    /* -- shape -- */
    int32_t n, sh_degree, width, height, tile_width, tile_height;
    int64_t capacity;        /* live pairs the list buffers hold (payload, records: fsgs_quad_stream_capacity(1, tw, th, capacity)) */
    /* -- parameters (read; stepped in place by launch 8) and the camera -- */
    float *means, *quats, *log_scales, *opac_logit, *features_dc, *features_rest;
    const float *viewmat, *K, *campos, *c2w, *background; /* [4,4] [3,3] [3] [3,4] as fsgs_sh_fwd_pack takes it, [3] */
    int32_t binarise; float binary_threshold;             /* dn_model.py:492-503 (the write happens in launch 1) */
    /* -- launch 1: projection outputs [frame], binning -- */
    float *scales_exp, *opac_sig; int32_t *radii; float *means2d, *depths, *conics;
    int32_t *tiles_per_gauss, *isect_offsets /* [T + 1] */;
    const int32_t *bucket_base /* [T + 1], the view's previous frame */; int32_t *tile_cursor /* [T], zero */;
    void *buckets /* [scratch] */; int64_t bucket_words; int32_t *next_bucket_base /* [T + 1] [frame] */;
    float growth; int32_t slack; int32_t *mapped /* (mapped) int32[4] */;
    float *packed /* [N,16] [scratch] */, *normals_world /* [N,3] [frame] */, *zero_cells; int32_t n_zero;
    int32_t *tile_order /* [T] [scratch] */;
    /* -- launch 2 -- */
    int32_t *payload /* [capacity] [frame] */, *long_flag /* nullable (a word inside zero_cells) */; int32_t rel_gate;
    /* -- launch 3: compositing forward (fsgs_raster_fwd_quad; walk = FSGS_WALK_ONE_WAVE) -- */
    float *render, *alphas; int32_t *last_ids; float *render_extra;          /* [frame] */
    float *records; int32_t *n_rec; float *seg_state; int32_t *seg_split;     /* [scratch] streams of the frame */
    float *max_last /* == zero_cells */;
    void *tail_scratch; int64_t tail_scratch_bytes; int32_t tail_items, handoff_records, handoff_rel_len; int64_t tail_epoch;
    int32_t *bwd_queue /* nullable */; int32_t bwd_queue_items;
    /* -- launch 4: images [frame] + the depth / normal L1 terms + the backward's dispatch order -- */
    float *rgb, *depth, *normal; int32_t n_cells;
    const float *gt_rgb, *gt_depth, *gt_normal /* nullable */, *seed /* [1]: d loss (1.0) */;
    float g_depth, g_normal; float *aux_partial, *v_depth_img, *v_normal_img /* nullable with gt_normal */;
    int32_t *order_counters /* nullable */, *bwd_order /* nullable */; int32_t order_shift;
    /* -- launches 5-6: SSIM + L1 on rgb, loss value -- */
    float *ssim_maps /* [3,H,W,3] */, *ssim_sums; int64_t ssim_rows, aux_rows;
    float g_l1, g_ssim, ssim_lambda; float *v_rgb, *loss_out /* [1] [frame] */;
    /* -- loss_kind = 1: get_loss_dict's default terms (dn_model.py:673-925 with FusionSense's switches: masked L1 + SSIM
     *    on rgb, EdgeAwareLogL1 / L1 / LogL1 / MSE + TV on the depth, L1 + TV on the normals, the min-scale term, the
     *    touch-normal MSE) instead of the benchmark loss: launch 4 then forms the images only, launch 5 is
     *    fsgs_ssim_l1_fwd_masked (gt_rgb = the view's image), one more launch — fsgs_fusion_aux_loss_riders (hook 8) —
     *    leaves the depth / normal gradient images (seed known) and the riders' partial sums, launch 6 is
     *    fsgs_ssim_l1_bwd_masked with the combine of all partial sums, and launch 8 carries min_scale_g.  gt_depth,
     *    g_depth, g_normal, aux_partial are not used.  (Mono depth, the cosine term and normals-from-depth keep the
     *    per-op route.) -- */
    int32_t loss_kind;
    const float *mask /* nullable [H,W] */, *sensor_depth /* [H,W] */;
    float depth_tol; float w_aux[7]; int32_t fa_flags;
    float *fa_partial; int64_t fa_rows;               /* [fa_rows, 8], fa_rows = fsgs_fusion_aux_num_partials(H, W) */
    float *ms_partial /* nullable: no min-scale term */; int64_t ms_rows; float g_min;
    int32_t n_touch; const int64_t *touch_idx; const float *touch_normals; float *touch_partial; int64_t touch_rows; float g_touch;
    /* -- launch 7: compositing backward -- */
    float *v_packed; int64_t replica_rows; int32_t dispatch_stride;
    /* -- launch 8: per-Gaussian backward + after_train statistics + Adam -- */
    float *absgrad /* [N,2] [frame] */, *xys_grad_norm, *vis_counts, *max_2Dsize /* nullable: no statistics */;
    float inv_max_hw; const uint8_t *frozen /* nullable */;
    fsgs_adam_groups adam; float min_scale_g; int32_t gsb_flags;
    /* adam.n_groups == 0: launch 8 is fsgs_gauss_sh_bwd instead — the parameter gradients are WRITTEN (a step without its
     * optimizer: gradient accumulation, callers that clip / log gradients, bench.py's figure without the optimizer), in
     * the layout of the parameters; with loss_kind 1 the min-scale term's gradient is then added by one more launch
     * (fsgs_min_scale_loss over ms_partial as scratch), as the per-op route does */
    float *g_means, *g_log_scales, *g_quats, *g_features_dc, *g_features_rest, *g_opac_logit;
    /* -- optional timing hooks: hipEvent_t handles (as void *) recorded on `stream` right before / behind launch k
     *    (k = 0..7 in the order above: project+bin, sorts, forward, epilogue, SSIM fwd | SSIM bwd, backward, per-Gaussian;
     *    k = 8: loss_kind 1's fsgs_fusion_aux_loss_riders, which runs behind launch 5);
     *    NULL = none.  A recorded event costs the GPU ~6 us of idle time in front of the next launch. -- */
    void *ev_before[9], *ev_after[9];
    /* -- written by the calls -- */
    int32_t armed;   /* 1 between fsgs_step_forward and fsgs_step_backward */
    int64_t wait_ns; /* fsgs_step_backward: host time spent waiting for the frame's verdict (the rest of a call is issue time) */
} fsgs_step_plan;
int fsgs_step_forward(fsgs_step_plan *plan, fsgs_stream_t stream);
int fsgs_step_backward(fsgs_step_plan *plan, int64_t spin_limit, int64_t *n_live_out, fsgs_stream_t stream);
int fsgs_step_run(fsgs_step_plan *plan, int64_t spin_limit, int64_t *n_live_out, fsgs_stream_t stream);
int64_t fsgs_step_plan_bytes(void); /* sizeof(fsgs_step_plan): a binding checks its own layout against it */

/* ---- semantic head: one layer, forward and backward -----------------------------------------------------------------
 * y = act(x W^T + b) + r.  x [rows, in] with rows `x_pitch` elements apart (0: one row for all), w [out, in] contiguous,
 * bias [out] nullable, residual [rows, out] (pitch res_pitch) nullable, y [rows, out] contiguous.  All of one element type;
 * products in that type on the matrix cores, sums fp32.  No pointer has to be aligned beyond its element; x, residual and dy
 * are read in 16-byte pieces between their first and last element, and a matrix of fewer bytes than that must have 16 readable. */
#define FSGS_F32 0
#define FSGS_BF16 1
#define FSGS_F16 2
#define FSGS_ACT_NONE 0
#define FSGS_ACT_RELU 1
#define FSGS_ACT_GELU 2 /* z/2 (1 + erf(z / sqrt 2)) */
#define FSGS_ACT_SILU 3
#define FSGS_LINEAR_MAX_DIM 65536
int fsgs_linear_fwd(int64_t rows, int in_dim, int out_dim, int dtype, const void *x, int64_t x_pitch, const void *w,
                    const void *bias, int act, const void *residual, int64_t res_pitch, void *y, fsgs_stream_t stream);
/* VJP.  dx [rows, in], dw [out, in], db [out]: contiguous, written, each nullable (rows == 0 writes nothing: dw and db are
 * the caller's to clear).  The pre-activation is formed again from x, w and bias.  The residual's gradient is dy itself.
 * y: nullable; the forward's output [rows, out] (contiguous) of a layer WITHOUT residual.  Where
 * fsgs_linear_bwd_uses_output says 1 (relu layers too wide for the one-pass kernel) its bits save that product: the forward
 * stores a positive value that rounds to zero as -0. */
int fsgs_linear_bwd_uses_output(int64_t rows, int in_dim, int out_dim, int dtype, int act);
int64_t fsgs_linear_bwd_scratch_bytes(int64_t rows, int in_dim, int out_dim, int dtype, int act, int want_dx, int want_dw,
                                      int want_db);
int fsgs_linear_bwd(int64_t rows, int in_dim, int out_dim, int dtype, const void *x, int64_t x_pitch, const void *w,
                    const void *bias, int act, const void *y, const void *dy, int64_t dy_pitch, void *dx, void *dw, void *db,
                    void *scratch, int64_t scratch_bytes, fsgs_stream_t stream);

/* ---- distillation from a teacher's top-K scores ---------------------------------------------------------------------
 * p = softmax over the row's K entries of teacher / T, q = softmax over all classes of logits / T,
 * L = T^2 sum_k p_k (log p_k - log q[idx_k]).  logits [rows, classes], idx [rows, K] (int32 or int64), teacher [rows, K]
 * (an element type of its own), weight [rows] nullable; rows `*_pitch` elements apart.  An entry whose class lies outside
 * [0, classes) is no entry; a class may stand in several entries.  Rows without entries, rows whose entries are all -inf and
 * rows of weight zero have loss and gradient zero and are not counted.
 *   reduction NONE: loss [rows] = weight L;  SUM: loss [1] = sum weight L;  MEAN: that over the sum of the weights.
 * stat [rows, 4] (16-byte aligned) and inv_weight [1] carry what the backward needs; both nullable when there is none.
 * scratch: fsgs_distill_scratch_bytes(), not used by NONE. */
#define FSGS_DISTILL_MAX_K 256
#define FSGS_DISTILL_MAX_CLASSES 524288 /* one bit per class in LDS */
#define FSGS_DISTILL_MIN_T 1e-6f /* temperature range: its square and its reciprocal stay normal numbers */
#define FSGS_DISTILL_MAX_T 1e6f
#define FSGS_REDUCE_NONE 0
#define FSGS_REDUCE_SUM 1
#define FSGS_REDUCE_MEAN 2
int64_t fsgs_distill_scratch_bytes(void);
int fsgs_distill_fwd(int64_t rows, int classes, int top_k, int dtype, const void *logits, int64_t pitch, int idx_bits,
                     const void *idx, int64_t idx_pitch, int teacher_dtype, const void *teacher, int64_t teacher_pitch,
                     const float *weight, float temperature, int reduction, float *loss, float *stat, float *inv_weight,
                     void *scratch, int64_t scratch_bytes, fsgs_stream_t stream);
/* grad_logits [rows, classes], contiguous, written.  grad_loss: [rows] when grad_per_row (reduction NONE), else [1];
 * inv_weight: what the forward left there (nullable: 1). */
int fsgs_distill_bwd(int64_t rows, int classes, int top_k, int dtype, const void *logits, int64_t pitch, int idx_bits,
                     const void *idx, int64_t idx_pitch, int teacher_dtype, const void *teacher, int64_t teacher_pitch,
                     const float *weight, float temperature, const float *stat, const float *inv_weight,
                     const float *grad_loss, int grad_per_row, void *grad_logits, fsgs_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* FSGS_H */
