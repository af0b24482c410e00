/*
 * doubletake_hip.h -- C ABI of the MI355X (gfx950) hot path for nianticlabs/doubletake.
 *
 * One shared library (doubletake_amd/_lib/libdoubletake_hip.so) exports everything below.
 * Conventions:
 *   - plain C linkage, raw DEVICE pointers + extents, no torch types;
 *   - every entry point takes the HIP stream to launch on (dt_stream_t == hipStream_t);
 *     nothing synchronises, nothing allocates device memory;
 *   - return 0 on success, non-zero on failure; dt_last_error() gives the message
 *     (thread-local).  Argument errors are detected before anything is launched.
 *   - tensors are dense fp32 unless the name says otherwise; "bchw" = NCHW, "bhwc" = NHWC.
 *
 * Each declaration cites the reference interface it replaces (paths relative to
 * /root/reference/src/doubletake/).  The reference has exactly one native ABI of its own
 * (tools/marching_cubes/ext.cpp:4-6); everything else it runs through torch ops, so for
 * those the "interface replaced" is the Python method whose body these kernels implement.
 * INTEGRATION.md shows the reference-side binding for every entry point.
 */
#ifndef DOUBLETAKE_HIP_H
#define DOUBLETAKE_HIP_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef void* dt_stream_t; /* hipStream_t */

/* ---- library ------------------------------------------------------------------------ */
/* ABI version: bumped whenever the signature of ANY entry point or a struct below changes (not for new entry points alone).
 * Bindings compare it with the version they were written against before the first call: an older .so called with
 * shifted arguments would corrupt device memory instead of failing.  History: 101 round 2; 102 round 3 (depth_planes /
 * channels arguments of dt_cv_lowest_cost_f32, dt_cv_overall_mask_u8, dt_cv_mlp_hint_simple_f32); 103 round 4;
 * 104 plan_scratch_bytes argument of dt_cv_mlp_hint_planned_f32; 105 the plan is written by dt_cv_mlp_plan_f32, the planned
 * call only consumes it; 106 dt_plane_desc.outside in the place of padding, which a caller could leave unset. */
#define DT_ABI_VERSION 106
int dt_version(void);
const char* dt_last_error(void);
/* number of HIP devices visible; <0 on runtime error.  No other call needs it. */
int dt_device_count(void);
/* Kernels launched by this library in this process so far (all streams, all entry points): lets a caller report the
 * launch count of a step as the difference of two reads (bench.py roofline_conv.launches). */
int64_t dt_kernel_launch_count(void);
/* A value that identifies the process-wide settings that change kernel selection or launch geometry (the plan objective mask
 * and the volume kernel's CU budget in force, whether preset by the environment or given to dt_conv_set_plan_objective /
 * dt_cv_mlp_set_cu_budget).  Replay mechanisms above the
 * ABI (captured hipGraphs, launch programs) bake those choices in; keying their caches on this token keeps a replay from
 * silently using the old ones, and setting a value back makes the old captures valid again. */
int64_t dt_settings_token(void);

/* ---- layout helpers (boundary between torch NCHW tensors and the kernels' NHWC) ------ */
int dt_nchw_to_nhwc_f32(const float* src, float* dst, int n, int c, int h, int w, dt_stream_t s);
int dt_nhwc_to_nchw_f32(const float* src, float* dst, int n, int c, int h, int w, dt_stream_t s);

/* ---- plane-sweep cost volume ---------------------------------------------------------
 * Parameter block written by dt_cv_setup_f32 and read by the volume kernels; per batch
 * element: [0..8] invK[:3,:3] row-major, [9..11] pad, [12..12+D) depth planes, then per
 * source view 20 floats: P = (K_src @ src_cam_T_cur_cam)[:3,:4] row-major (12),
 * t_src = cur_cam_T_src_cam[:3,3] (3), pose_dist, R_measure, t_measure (3), pad (2).
 */
int dt_cv_params_floats(int num_planes, int num_src); /* floats per batch element */

/* replaces: CostVolumeManager.generate_depth_planes (modules/cost_volume.py:96-130),
 * Project3D's P = K @ cam_T_world (utils/geometry_utils.py:82), pose_distance
 * (utils/geometry_utils.py:187-199). */
int dt_cv_setup_f32(const float* src_Ks_bk44, const float* src_extrinsics_bk44,
                    const float* src_poses_bk44, const float* cur_invK_b44,
                    const float* min_depth_b, const float* max_depth_b,
                    int batch, int num_src, int num_planes, float* params_out, dt_stream_t s);

/* replaces: the two torch.matmul calls on the tuple's 4x4 camera matrices in DepthModelCVHint.forward
 * (experiment_modules/doubletake_model.py:330-339): src_cam_T_cur_cam[b,k] = src_cam_T_world[b,k] @ cur_world_T_cam[b] and
 * cur_cam_T_src_cam[b,k] = cur_cam_T_world[b] @ src_world_T_cam[b,k], fp32, row-major 4x4, in one launch. */
int dt_cv_relative_poses_f32(const float* src_cam_T_world_bk44, const float* src_world_T_cam_bk44,
                             const float* cur_cam_T_world_b44, const float* cur_world_T_cam_b44, int batch, int num_src,
                             float* src_cam_T_cur_cam_bk44, float* cur_cam_T_src_cam_bk44, dt_stream_t s);
/* replaces: CostVolumeManager.warp_features (modules/cost_volume.py:132-217) as a stand-alone op: warp every
 * source view to the current view at ONE depth map per batch element.  src NCHW [b,k,c,h,w]; params from
 * dt_cv_setup_f32 (num_planes = the D it was built with); outputs: world points [b*k,4,h*w], projected depths
 * [b,k,h,w] (z + 1e-8), warped features [b,k,c,h,w], mask [b,k,h,w] (1.0 where depth > 0).  The fused volume
 * kernels do not use it. */
int dt_cv_warp_f32(const float* src_bkchw, const float* params, const float* depth_bhw, int batch,
                   int num_src, int channels, int h, int w, int num_planes, float* world_points_B4N,
                   float* depths_bkhw, float* warped_bkchw, float* mask_bkhw, dt_stream_t s);
/* replaces: CostVolumeManager.build_cost_volume (modules/cost_volume.py:219-315)
 * = warp_features (:132-217) + channel dot + z'>0 mask + sum over views.
 * src_feats_bkhwc is NHWC (use dt_nchw_to_nhwc_f32 with n = b*k).  volume_bdhw is NCHW. */
int dt_cv_dot_f32(const float* cur_feats_bchw, const float* src_feats_bkhwc, const float* params,
                  float* volume_bdhw, int batch, int num_src, int channels, int h, int w,
                  int num_planes, dt_stream_t s);
/* dt_cv_dot_f32 stages each source view's footprint of a pixel tile in LDS (csrc/cv_dot_lds.hip).  Two companions of
 * the same kernel, for parity tests and ablations: ..._direct_ samples every tap straight from global memory (same
 * expressions in the same order: bit-identical volume); ..._stats_ additionally counts, in stats4[0..3] (device ints,
 * zeroed by the caller), (tile, plane-range, view) units that were staged / took the direct path / saw nothing of the
 * view, and individual taps that missed their staged box (expected 0). */
int dt_cv_dot_direct_f32(const float* cur_feats_bchw, const float* src_feats_bkhwc, const float* params,
                         float* volume_bdhw, int batch, int num_src, int channels, int h, int w,
                         int num_planes, dt_stream_t s);
int dt_cv_dot_stats_f32(const float* cur_feats_bchw, const float* src_feats_bkhwc, const float* params,
                        float* volume_bdhw, int batch, int num_src, int channels, int h, int w,
                        int num_planes, int* stats4, dt_stream_t s);

/* replaces: FeatureVolumeManager.build_cost_volume (modules/feature_volume.py:81-356) and
 * FeatureMeshHintVolumeManager.build_cost_volume (modules/mesh_hint_volume.py:84-393; Fast
 * variant :679-928): warp + metadata + 202->128->128->1 matching MLP (+ 3->12->12->1 hint
 * MLP when hint_mlp != NULL), fused, fp32 MFMA.
 *   w1dyn/w1pix/w2p/tail: matching-MLP weights re-packed for the kernel's K order by
 *     doubletake_amd.modules.mlp_pack (sizes from dt_cv_mlp_pack_floats);
 *   hint_mlp: 217 floats = V1[12x3], c1[12], V2[12x12], c2[12], V3[12], c3 (nn.Linear
 *     layouts, row-major) or NULL;
 *   depth_hint / hint_weights / hint_mask: [b,1,hint_h,hint_w] maps (NaN allowed where mask==0),
 *     ignored when hint_mlp == NULL;
 *   out_nhwc: 0 -> volume [b,D,h,w]; 1 -> [b,h,w,D] (torch channels_last of the same tensor);
 *   num_src: 1..15 source views -- up to 7 (the reference default) every view's layer-1 weights stay resident in LDS, the
 *     views beyond the seventh read theirs from L2 inside the view loop.
 */
int dt_cv_mlp_pack_floats(int num_src, int* w1dyn, int* w1pix, int* w2p, int* tail);
int dt_cv_mlp_hint_f32(const float* cur_feats_bchw, const float* src_feats_bkhwc,
                       const float* params, const float* w1dyn, const float* w1pix,
                       const float* w2p, const float* tail, const float* hint_mlp,
                       const float* depth_hint_b1HW, const float* hint_weights_b1HW,
                       const float* hint_mask_b1HW, int hint_h, int hint_w, float* volume,
                       int out_nhwc, int batch, int num_src, int h, int w, int num_planes,
                       dt_stream_t s);
/* dt_cv_mlp_hint_f32 with a COST-AWARE SPAN PLAN (round 4).  The hint kernel skips the feature contractions of views a pixel
 * tile cannot see, so its (tile, plane) units differ in cost; dt_cv_mlp_plan_f32 prices every unit by the number of source views
 * it can see (two small launches that read only `params`, i.e. the cameras and planes) and writes the unit at which every wave's
 * span of equal estimated work begins; dt_cv_mlp_hint_planned_f32 runs the volume kernel on those spans.  Same volume as
 * dt_cv_mlp_hint_f32 (the plan only moves span boundaries).  A plan depends on (params, batch, num_src, h, w, num_planes) and
 * the device: it may be reused for further calls with the same cameras.
 * plan_scratch: device buffer of at least dt_cv_mlp_plan_bytes(batch, h, w, num_planes) bytes (for the device that is current at
 * the call), owned by the caller; its size is passed and checked by both calls (a scratch sized for another shape or device is
 * refused, not overrun).  dt_cv_mlp_hint_planned_f32 must be given a scratch that dt_cv_mlp_plan_f32 filled for the same
 * arguments earlier on the same stream (or ordered before it); where the plan does not apply (more source views than the kernel
 * keeps in LDS, DT_MLP_PLAN=0) dt_cv_mlp_plan_f32 launches nothing and the planned call uses equal-length spans. */
int64_t dt_cv_mlp_plan_bytes(int batch, int h, int w, int num_planes);
/* Compute-unit budget of the fused volume kernel (round 5: spatial partition of the chip).  The kernel is persistent -- one
 * workgroup per compute unit, each owning the whole unit (all of its LDS and registers) -- so with several keyframes in flight
 * it alternates with the latency-bound conv stacks of the other frames instead of running beside them.  With a budget of
 * `cus` (> 0, rounded down to a multiple of 8 but never below 8, at most the device's count; 0 = the whole device, the default) every later
 * dt_cv_mlp_plan_f32 / dt_cv_mlp_hint*_f32 call launches only that many workgroups, leaving the other compute units to kernels of
 * other streams for the whole launch.  Same volume (the budget only changes how the (tile, plane) units are dealt to waves).
 * Process-wide; set it before a plan is written, and do not change it between dt_cv_mlp_plan_f32 and the planned call that
 * consumes the plan.  Returns the budget now in force. */
int dt_cv_mlp_set_cu_budget(int cus);
int dt_cv_mlp_plan_f32(const float* params, int batch, int num_src, int h, int w, int num_planes, void* plan_scratch,
                       int64_t plan_scratch_bytes, dt_stream_t s);
int dt_cv_mlp_hint_planned_f32(const float* cur_feats_bchw, const float* src_feats_bkhwc,
                               const float* params, const float* w1dyn, const float* w1pix,
                               const float* w2p, const float* tail, const float* hint_mlp,
                               const float* depth_hint_b1HW, const float* hint_weights_b1HW,
                               const float* hint_mask_b1HW, int hint_h, int hint_w, float* volume,
                               int out_nhwc, int batch, int num_src, int h, int w, int num_planes,
                               const void* plan, int64_t plan_bytes, dt_stream_t s);
/* OPT-IN split-precision variant of dt_cv_mlp_hint_f32 (same reference functions, same arguments except the weights):
 * the two dense contractions run on v_mfma_f32_32x32x16_f16 with every operand split into fp16 hi + lo parts
 * (x*w ~= x_hi*w_hi + x_lo*w_hi + x_hi*w_lo, fp32 accumulation): fp32-class accuracy (dropped term 2^-22 relative) at 3/16
 * of the fp32 matrix time.  Not the default anywhere.  Requires |inputs|, |weights|, |activations| < 65504.
 * w1dyn/w1pix/w2: uint16 arrays of fp16 fragments from doubletake_amd.modules.mlp_pack.pack_mlp_split (sizes from
 * dt_cv_mlp_split_pack_halves); tail: the same 260 floats as the fp32 kernel. */
int dt_cv_mlp_split_pack_halves(int num_src, int* w1dyn, int* w1pix, int* w2);
int dt_cv_mlp_hint_split_f32(const float* cur_feats_bchw, const float* src_feats_bkhwc, const float* params,
                             const uint16_t* w1dyn_h, const uint16_t* w1pix_h, const uint16_t* w2_h, const float* tail,
                             const float* hint_mlp, const float* depth_hint, const float* hint_weights,
                             const float* hint_mask, int hint_h, int hint_w, float* volume, int out_nhwc, int batch,
                             int num_src, int h, int w, int num_planes, dt_stream_t s);

/* Same function, one thread per (pixel, plane), plain fp32 FMAs, nn.Linear weight layouts
 * (W1 [128,Cin], b1, W2 [128,128], b2, W3 [1,128], b3; Cin = (channels + 4)(num_src + 1) + 6 num_src,
 * modules/feature_volume.py:49-67).  GPU-side cross-check of the fused kernel in the parity tests, and the
 * product path for the shapes the fused kernel does not take: matching_dim_size != 16 (channels <= 32), more
 * than 15 source views (<= 16), and caller-supplied per-pixel depth planes -- depth_planes_bdhw [b,D,h,w] or
 * null (modules/mesh_hint_volume.py:95,149-150,211: "optionally, provide a depth plane to use instead of
 * constructing one here"). */
int dt_cv_mlp_hint_simple_f32(const float* cur_feats_bchw, const float* src_feats_bkhwc,
                              const float* params, const float* depth_planes_bdhw, const float* W1,
                              const float* b1, const float* W2, const float* b2, const float* W3,
                              const float* b3, const float* hint_mlp,
                              const float* depth_hint_b1HW, const float* hint_weights_b1HW,
                              const float* hint_mask_b1HW, int hint_h, int hint_w,
                              float* volume_bdhw, int batch, int num_src, int channels, int h, int w,
                              int num_planes, dt_stream_t s);

/* CostVolumeManager.build_cost_volume (modules/cost_volume.py:219-315) one thread per (pixel, plane): any
 * channel count, depth_planes_bdhw [b,D,h,w] or null (:249-250).  dt_cv_dot_f32 is the tuned kernel for
 * 16 channels and one plane list per batch element. */
int dt_cv_dot_simple_f32(const float* cur_feats_bchw, const float* src_feats_bkhwc, const float* params,
                         const float* depth_planes_bdhw, float* volume_bdhw, int batch, int num_src,
                         int channels, int h, int w, int num_planes, dt_stream_t s);

/* replaces: argmax + gather in CostVolumeManager.forward (modules/cost_volume.py:355-361).
 * volume may be NCHW (nhwc = 0) or NHWC (nhwc = 1); first maximum wins.  The returned depth is
 * depth_planes_bdhw's entry at the pixel when that tensor is given (indices_to_disparity's gather, :317-320),
 * the parameter block's plane list otherwise. */
int dt_cv_lowest_cost_f32(const float* volume, const float* params, const float* depth_planes_bdhw,
                          float* lowest_bhw, int nhwc, int batch, int num_src, int h, int w,
                          int num_planes, dt_stream_t s);

/* replaces: get_mask + depth mask at the LAST plane (modules/cost_volume.py:73-94,
 * modules/mesh_hint_volume.py:270-287 [per_view = 1 -> uint8 [b,k,h,w]] and :818-822
 * [per_view = 0 -> uint8 [b,h,w]]); depth_planes_bdhw as above. */
int dt_cv_overall_mask_u8(const float* params, const float* depth_planes_bdhw, uint8_t* mask_out,
                          int per_view, int batch, int num_src, int h, int w, int num_planes,
                          dt_stream_t s);

/* ---- the volume as a distribution over depth planes ------------------------------------
 * The D plane scores of a pixel read as logits.  With y_d = scale * x_d over the planes the mask leaves visible, m = max x and
 * s = sum_d exp(scale (x_d - m)):
 *   log_sum = scale m + ln s;   lp_d = scale (x_d - m) - ln s;   entropy = -sum_d exp(lp_d) lp_d
 * No reference counterpart: dt_cv_lowest_cost_f32's argmax (modules/cost_volume.py:355-361) is the most probable plane of the same
 * distribution.  Statistics are fp32 whatever the volume's type.  Edges, the same for every entry point below:
 *   - masked planes may hold anything (NaN, infinities); a score of -inf is a plane without probability;
 *   - a pixel without any probability: log_sum = log_prob = -inf, entropy = 0, no alternatives, gradient 0;
 *   - a visible NaN or +inf makes the pixel's real-valued outputs NaN (the order of the alternatives stays defined: NaN first);
 *   - a given plane outside 0..d-1 scores nothing: log_prob = dt_plane_desc.outside, no gradient;
 *   - equal scores: the lowest plane first; alternatives beyond the planes with probability: plane -1, log prob -inf, depth 0. */
enum { DT_VOL_F32 = 0, DT_VOL_F16 = 1, DT_VOL_BF16 = 2 };
#define DT_PLANE_MAX_TOP 8
#define DT_PLANE_MAX_PLANES (1 << 16)  /* of a volume: what float32 sums over the planes bear (ln s within 1e-3) */
#define DT_PLANE_MAX_NEAREST (1 << 30) /* of dt_cv_nearest_planes_f32, which sums nothing */

typedef struct dt_plane_desc {
  int b, d, h, w;             /* extents of the volume; b * h * w < 2^31 - 1, d <= DT_PLANE_MAX_PLANES */
  int dtype;                  /* DT_VOL_*: type of the volume and of its gradient */
  int top;                    /* alternatives per pixel, 0..min(d, DT_PLANE_MAX_TOP) */
  float scale;                /* inverse temperature, 1e-30..1e30 */
  float outside;              /* log_prob where the given plane is outside 0..d-1: 0 for losses, -inf where certainty is asked for */
  int64_t vol_stride[4];      /* elements between neighbours along b, d, y, x: any layout, none negative */
  int64_t mask_stride[4];     /* bytes, likewise; 0 along a broadcast axis */
  int64_t planes_stride[4];   /* elements of the depth planes, likewise */
  int64_t grad_stride[4];     /* elements of the gradient written by ..._grad; the other call ignores it */
} dt_plane_desc;

/* Statistics of every pixel in one pass over the volume.  mask (1 byte per plane, 0 = not visible), plane_bhw and depth_planes may
 * be NULL; depth_planes is read for the alternatives' depths only.  Outputs are dense; entropy and log_sum [b,h,w] are always
 * written.  log_prob [b,h,w] goes with plane_bhw: both or neither.  With top > 0 top_log_prob and top_plane [b,top,h,w] are both
 * required; top_depth [b,top,h,w] may be NULL and needs depth_planes.  row_max and row_log [b,h,w], both or neither, are m and
 * ln s, what ..._grad needs. */
int dt_cv_plane_log_probs(const dt_plane_desc* d, const void* volume, const uint8_t* mask, const int64_t* plane_bhw,
                          const float* depth_planes, float* log_prob, float* entropy, float* log_sum, float* top_log_prob,
                          int64_t* top_plane, float* top_depth, float* row_max, float* row_log, dt_stream_t s);
/* Gradient of the volume for gradients of the outputs above (each NULL where there is none; dense, shaped like its output):
 *   dx_d = scale [ sum of the gradients that meet plane d (given plane, alternatives)
 *                  + p_d (g_log_sum - g_log_prob - sum g_top) - g_entropy p_d (lp_d + entropy) ]
 * mask, plane_bhw, entropy, top_plane, row_max and row_log are those of the forward call; g_log_prob needs plane_bhw, g_top_log_prob
 * needs top_plane, without them either may be NULL.  Every element of the gradient is written (0 for masked planes and scores of
 * -inf). */
int dt_cv_plane_log_probs_grad(const dt_plane_desc* d, const void* volume, const uint8_t* mask, const int64_t* plane_bhw,
                               const float* entropy, const int64_t* top_plane, const float* row_max, const float* row_log,
                               const float* g_log_prob, const float* g_entropy, const float* g_log_sum, const float* g_top_log_prob,
                               void* grad_volume, dt_stream_t s);
/* The plane a metric depth falls on: argmin_d |depth - planes_d| per pixel, the lowest plane of equal ones.  Differences are taken in
 * 64 bits: exact for planes within a factor of 2^29 of the depth, rounded beyond, so that planes whose distances differ by less than
 * a step of 64 bits count as equally near (a depth of 1e20 is equally far from all planes of a few metres: plane 0).  -1 where the
 * depth is not finite or not positive.  depth dense [b,h,w]; planes read through planes_stride4 (b, d, y, x; 0 along a broadcast
 * axis, none negative), at most DT_PLANE_MAX_NEAREST; a plane that is no finite number is never the nearest. */
int dt_cv_nearest_planes_f32(const float* depth_bhw, const float* depth_planes, const int64_t* planes_stride4, int b, int d, int h,
                             int w, int64_t* plane_bhw, dt_stream_t s);

/* ---- conv stacks (cost-volume encoder / depth decoders) --------------------------------
 * One implicit-GEMM primitive on NHWC fp32 tensors (fp32 MFMA):
 *   out[n,y,x,co] = act( bias[co] + sum_{ky,kx,ci} W[co,ky,kx,ci] * in[n, y*stride+ky-pad,
 *                   x*stride+kx-pad, ci] (+ residual[n,y,x,co]) )
 * where `in` is the virtual channel-concatenation of up to three NHWC sources, each
 * optionally nearest-upsampled x2 on the fly.  Replaces nn.Conv2d + bias + LeakyReLU/ELU +
 * residual add + torch.cat + F.interpolate(nearest) as composed in BasicBlock
 * (modules/layers.py:77-94), CVEncoder.forward (modules/networks.py:110-117),
 * ConvBlock / ConvUpsampleAndConcatBlock (modules/networks_fast.py:17-40).
 * Weights are pre-packed by doubletake_amd.modules.conv_pack (dt_conv_pack_floats).
 */
enum { DT_ACT_NONE = 0, DT_ACT_LRELU02 = 1, DT_ACT_ELU = 2, DT_ACT_RELU = 3 };

typedef struct dt_conv_desc {
  int n, h_out, w_out;      /* output extent */
  int c_out;                /* multiple of 32 */
  int nsrc;                 /* 1..3 sources, concatenated along channels in order */
  int c[3];                 /* channels of each source (multiples of 8) */
  int up[3];                /* 1: source is (h_in/2, w_in/2) and read nearest-upsampled x2 */
  int ksize;                /* 1 or 3 (pad = ksize/2) */
  int stride;               /* 1 or 2 */
  int act;                  /* DT_ACT_* */
  int h_in, w_in;           /* extent of the (virtual, post-upsample) input */
  int pad_mode;             /* 0: zero padding; 1: replicate (nn.Conv2d padding_mode="replicate") */
  int transposed;           /* 1: tile the image with tall 8x4 instead of 4x8 output patches (fewer partly empty tiles
                             * on maps such as 15x20); packed_w must then come from the weight with its two spatial
                             * axes swapped (W.transpose(2,3)).  Extents above stay the real ones, results are the
                             * same.  Only where dt_conv_transposed_tiling() returns 1; 0 everywhere else. */
} dt_conv_desc;

int64_t dt_conv_pack_floats(int c_out, int c_in, int ksize);
/* W_oihw: nn.Conv2d weight [c_out, c_in, k, k] (device); packed: device buffer of
 * dt_conv_pack_floats floats. */
int dt_conv_pack_f32(const float* W_oihw, float* packed, int c_out, int c_in, int ksize,
                     dt_stream_t s);
int dt_conv2d_f32(const dt_conv_desc* d, const float* in0, const float* in1, const float* in2,
                  const float* packed_w, const float* bias, const float* residual,
                  float* out, dt_stream_t s);
/* 1 when dt_conv2d_f32 / dt_conv2d_pair_f32 (direct kernels) would run this convolution with fewer workgroups in the
 * transposed tiling (d->transposed is ignored on input); the caller then sets d->transposed = 1 and passes weights packed
 * from W.transpose(2,3). */
int dt_conv_transposed_tiling(const dt_conv_desc* d);
/* Plan objective of the conv launchers (round 5).  0 (default) = latency: a layer that cannot fill the chip splits its K loop over
 * 8 waves and / or several workgroups so that ONE launch on an idle chip finishes as early as possible.  With several
 * independent frames in flight (streams) that buys latency with resources another stream's kernels could use: a bit mask
 * switches the individual choices off -- 1: Winograd layers keep 256-thread workgroups (no in-workgroup K split); 2: direct 3x3
 * K-split kernels use 4 waves instead of 8; 4: no K split across workgroups; 8: no tail split; 16: low-resolution 1x1
 * convolutions on the plain kernel.  DT_CONV_THROUGHPUT below is the combination measured best with 4 keyframes in flight.
 * Results are unchanged up to the fp32 summation order of the K splits (same products).  Process-wide; returns the mask in force. */
#define DT_CONV_LATENCY 0
#define DT_CONV_THROUGHPUT 11
int dt_conv_set_plan_objective(int mask);
/* Winograd F(2x2,3x3) variant for 3x3 stride-1 convolutions (2.25x fewer multiplies; same fp32
 * arithmetic type, different summation order: results agree with dt_conv2d_f32 to ~1e-6 relative).
 * packed_w: dt_conv_wino_pack_floats floats made by dt_conv_wino_pack_f32 from the OIHW weight. */
int64_t dt_conv_wino_pack_floats(int c_out, int c_in);
int dt_conv_wino_pack_f32(const float* W_oihw, float* packed, int c_out, int c_in, dt_stream_t s);
int dt_conv2d_wino_f32(const dt_conv_desc* d, const float* in0, const float* in1, const float* in2,
                       const float* packed_w, const float* bias, const float* residual,
                       float* out, dt_stream_t s);
/* OPT-IN split-precision Winograd variant (csrc/conv_wino_split.hip): same function as dt_conv2d_wino_f32, the Winograd-domain
 * products as fp16 hi/lo pairs on v_mfma_f32_32x32x16_f16 with fp32 accumulation (x*w ~= x_hi*w_hi + x_lo*w_hi + x_hi*w_lo,
 * 2^-22 relative).  Not the default path.  Needs every source to be a multiple of 16 channels (..._supported returns 1).
 * packed_w: dt_conv_wino_split_pack_halves 16-bit words made by dt_conv_wino_split_pack_f16 from the OIHW weight. */
int64_t dt_conv_wino_split_pack_halves(int c_out, int c_in);
int dt_conv_wino_split_pack_f16(const float* W_oihw, uint16_t* packed, int c_out, int c_in, dt_stream_t s);
int dt_conv2d_wino_split_supported(const dt_conv_desc* d);
int dt_conv2d_wino_split_f32(const dt_conv_desc* d, const float* in0, const float* in1, const float* in2,
                             const uint16_t* packed_w, const float* bias, const float* residual,
                             float* out, dt_stream_t s);
/* conv1 and the shortcut ("downsample") conv of a BasicBlock (modules/layers.py:77-94) in ONE launch: both read the
 * same (virtually concatenated) sources.  A: 3x3, stride 1 or 2, weights packed by dt_conv_wino_pack_f32 when a_wino != 0
 * (stride 1 only) else by dt_conv_pack_f32.  B: 1x1 stride 1 (with a stride-1 A) or 3x3 stride 2 (with a stride-2 A),
 * weights packed by dt_conv_pack_f32.  da->act / db->act are applied per convolution; no residual inputs.  Kernel
 * pairs without a common workgroup size are issued as two launches inside the call. */
int dt_conv2d_pair_f32(const dt_conv_desc* da, const dt_conv_desc* db, const float* in0, const float* in1, const float* in2,
                       const float* packed_wa, int a_wino, const float* bias_a, float* out_a, const float* packed_wb,
                       const float* bias_b, float* out_b, dt_stream_t s);
/* direct (one thread per output element) version of the same primitive taking the
 * unpacked nn.Conv2d weight; GPU-side cross-check for the parity tests. */
int dt_conv2d_simple_f32(const dt_conv_desc* d, const float* in0, const float* in1,
                         const float* in2, const float* W_oihw, const float* bias,
                         const float* residual, float* out, dt_stream_t s);
/* 1x1 conv to ONE output channel (regression heads: modules/networks.py:60-63,
 * modules/networks_fast.py:102-132 last layer).  in NHWC [n,h,w,c] -> out [n,h,w].
 * out_exp (may be NULL): also receives expf(out), the depth of a log-depth head
 * (experiment_modules/doubletake_model.py:410-418) without a second pass. */
int dt_conv1x1_head_f32(const float* in_nhwc, const float* w_c, const float* bias1,
                        float* out, float* out_exp, int64_t pixels, int c, dt_stream_t s);
/* Fused regression head of the small decoder: per pixel Cin -> 128 (ELU) -> 128 (ELU) -> 1, i.e. the
 * three 1x1 convs of SkipDecoderRegression.out{1..4} (modules/networks_fast.py:102-132,134-141) in
 * one kernel.  cin = 64 or 128; wa/wb/tail packed by doubletake_amd.modules.mlp_pack.pack_head_mlp
 * (sizes from dt_head_mlp_pack_floats).  in NHWC [pixels][cin] -> out [pixels]. */
int dt_head_mlp_pack_floats(int cin, int* wa, int* wb, int* tail);
int dt_head_mlp_f32(const float* in_nhwc, const float* wa, const float* wb, const float* tail,
                    float* out, float* out_exp, int64_t pixels, int cin, dt_stream_t s);
/* The same head for up to 4 independent feature maps (the coarse scales of one decoder pass,
 * modules/networks_fast.py:134-141 loops over them) in ONE launch.  Host-side tables of n_heads device
 * pointers / sizes; every map at most 32768 pixels; out_exp (table or entries) may be NULL.  Results are
 * bit-identical to n_heads calls of dt_head_mlp_f32. */
int dt_head_mlp_multi_f32(int n_heads, const float* const* in_nhwc, const float* const* wa,
                          const float* const* wb, const float* const* tail, float* const* out,
                          float* const* out_exp, const int64_t* pixels, const int* cin, dt_stream_t s);
/* dt_conv2d_wino_f32 and dt_head_mlp_multi_f32 in ONE launch (round 5): SkipDecoderRegression's heads of scales 3, 2, 1
 * (modules/networks_fast.py:134-141) depend on decoder features that are final before the last block's 240x320 convolutions
 * start, and nothing depends on them, so their workgroups ride at the END of that convolution's grid (the shipped order, DT_HEADS_FIRST=0: they start as the conv's first round of workgroups drains; in front of the conv blocks measured slower) instead of waiting at
 * the end of the stream as a launch of their own (one workgroup's dependent MFMA chain long).  Arguments: those of the two
 * calls.  Only chip-filling Winograd launches (>= 2 workgroups per CU) are fused; anything else runs as the two launches.
 * Results are bit-identical to the two launches. */
int dt_conv2d_wino_heads_f32(const dt_conv_desc* d, const float* in0, const float* in1, const float* in2,
                             const float* packed_w, const float* bias, const float* residual, float* out,
                             int n_heads, const float* const* head_in_nhwc, const float* const* head_wa,
                             const float* const* head_wb, const float* const* head_tail, float* const* head_out,
                             float* const* head_out_exp, const int64_t* head_pixels, const int* head_cin,
                             dt_stream_t s);
/* bilinear x2 upsample, align_corners=False (utils/generic_utils.py:95-104), NHWC. */
int dt_upsample2x_bilinear_f32(const float* in_nhwc, float* out_nhwc, int n, int h, int w,
                               int c, dt_stream_t s);
/* exp() of the log-depth heads (experiment_modules/doubletake_model.py:410-418). */
int dt_exp_f32(const float* in, float* out, int64_t count, dt_stream_t s);

/* ---- matching encoder (next row of the path: modules/networks.py:138-189) -----------------
 * The convolutions run on dt_conv2d_f32 (BatchNorm folded into weight/bias on the host, ReLU as
 * DT_ACT_RELU, the final 3x3 with pad_mode = 1); these are the ops between them.  NHWC fp32. */
/* 7x7 stride-2 pad-3 stem conv as im2col: image NCHW [n,3,H,W] -> cols [n,Ho,Wo,152] with column
 * ci*49+ky*7+kx (= weight.reshape(c_out,-1) order), columns 147..151 zero; Ho=(H-1)/2+1. */
int dt_stem_im2col_f32(const float* image_nchw, float* cols_nhwc, int n, int H, int W, dt_stream_t s);
/* The same conv fused (no im2col buffer): image NCHW [n,3,H,W] -> out NHWC [n,Ho,Wo,64] with bias
 * (folded BatchNorm) and DT_ACT_RELU/NONE.  packed_w: dt_stem_pack_floats() floats made by
 * dt_stem_pack_f32 from the [64,3,7,7] weight (device pointers). */
int dt_stem_pack_floats(void);
int dt_stem_pack_f32(const float* W_64x3x7x7, float* packed, dt_stream_t s);
int dt_stem_conv_f32(const float* image_nchw, const float* packed_w, const float* bias64,
                     float* out_nhwc, int n, int H, int W, int act, dt_stream_t s);
/* nn.MaxPool2d(ksize, stride, pad) (torchvision resnet: 3,2,1; anti-aliased resnet: 2,1,0). */
int dt_maxpool_f32(const float* in_nhwc, float* out_nhwc, int n, int h, int w, int c, int ksize,
                   int stride, int pad, dt_stream_t s);
/* BlurPool(filt_size=4, stride=2, reflect pad (1,2,1,2)) of anti-aliased ResNets: depthwise 4x4
 * filter filt16 (HOST pointer, row-major; the module's `filt` buffer), ho=(h-1)/2+1. */
int dt_blurpool4_s2_f32(const float* in_nhwc, float* out_nhwc, const float* filt16_host, int n, int h,
                        int w, int c, dt_stream_t s);
/* MaxPool2d(2, stride 1) followed by that BlurPool, fused (one read of the input):
 * in [n,h,w,c] -> out [n,(h-2)/2+1,(w-2)/2+1,c]. */
int dt_maxblur_f32(const float* in_nhwc, float* out_nhwc, const float* filt16_host, int n, int h,
                   int w, int c, dt_stream_t s);
/* nn.InstanceNorm2d(c) (affine=False, biased variance) + optional LeakyReLU(0.2).  in NHWC with
 * c_stride >= c floats per pixel (only the first c are normalised); out [n,hw,c] or, with
 * out_nchw, [n,c,hw].  workspace: dt_instnorm_workspace_bytes(n,hw,c) device bytes. */
int64_t dt_instnorm_workspace_bytes(int n, int hw, int c);
int dt_instnorm_f32(const float* in_nhwc, float* out, void* workspace, int n, int hw, int c,
                    int c_stride, float eps, int act, int out_nchw, dt_stream_t s);

/* ---- TSDF fusion -----------------------------------------------------------------------
 * Volume: values/weights fp16 [X,Y,Z] (Z fastest), voxel (i,j,k) centre =
 * half(float(origin) + (i,j,k)*voxel_size) as in TSDF.generate_voxel_coords
 * (tools/tsdf.py:157-166).  `active` is a bitmap of X*Y*Z bits (uint32 words, bit id&31 of word
 * id>>5, id = (i*Y + j)*Z + k) replacing the open3d HashSet of active voxel keys
 * (tools/tsdf.py:79-84,530-538).  uint16_t* = IEEE half bits.
 */
int dt_tsdf_frame_params_floats(void);
/* replaces the per-frame prologue of TSDFFuser.integrate_depth (tools/tsdf.py:446-455):
 * inverse of K and cam_T_world (fp32 -> half), get_frustum_bounds (:15-50), P = K @ T (:407).
 * K16_44 / T16_44: device, 16 halves each.  frame_params: device, dt_tsdf_frame_params_floats. */
int dt_tsdf_frame_setup_f16(const uint16_t* K16_44, const uint16_t* T16_44, int img_h, int img_w,
                            float depth_min, float depth_max, float* frame_params, dt_stream_t s);

/* scalar thresholds of one fuser, prepared on the host with the reference's rounding points
 * (doubletake_amd/tools/tsdf.py: trunc = fp32(3*vs); thr_neg = half(-trunc [*1.5]);
 * thr_pos = half(trunc); max_depth_h = half(max_depth); depth_range = fp32(max - min)). */
typedef struct dt_tsdf_thresholds {
  float trunc, thr_neg, thr_pos, max_depth_h, min_depth, depth_range;
} dt_tsdf_thresholds;

/* replaces: the per-voxel body of TSDFFuser.integrate_depth for ONE frame (tools/tsdf.py:457-558)
 * incl. project_to_camera (:401-412); fp16-faithful (one rounding per reference op).
 * origin3: HOST pointer to the 3 fp32 origin components; depth_hw_f16: device [img_h,img_w]. */
int dt_tsdf_integrate_f16(uint16_t* values, uint16_t* weights, uint32_t* active,
                          const float* origin3, float voxel_size, int X, int Y, int Z,
                          const uint16_t* depth_hw_f16, int img_h, int img_w,
                          const float* frame_params, const dt_tsdf_thresholds* th, dt_stream_t s);
/* Batched forms: num_frames frames in ONE launch each.  K16/T16: [num_frames,16] halves;
 * frame_params: [num_frames, dt_tsdf_frame_params_floats()]; depth: [num_frames,img_h,img_w].
 * Frames are applied in index order per voxel (the reference's batch loop, tools/tsdf.py:440-445),
 * so the result is bit-identical to num_frames single-frame calls; the voxel is read and written
 * once instead of once per frame. */
int dt_tsdf_frames_setup_f16(const uint16_t* K16, const uint16_t* T16, int num_frames, int img_h,
                             int img_w, float depth_min, float depth_max, float* frame_params,
                             dt_stream_t s);
int dt_tsdf_integrate_frames_f16(uint16_t* values, uint16_t* weights, uint32_t* active,
                                 const float* origin3, float voxel_size, int X, int Y, int Z,
                                 const uint16_t* depth_f16, int num_frames, int img_h, int img_w,
                                 const float* frame_params, const dt_tsdf_thresholds* th,
                                 dt_stream_t s);
/* the same with fp32 depth maps, rounded to half inside the kernel exactly as fuse_frames' .half() would
 * (tools/fusers_helper.py:67-73): saves the converting copy in front of every integration */
int dt_tsdf_integrate_frames_f32depth_f16(uint16_t* values, uint16_t* weights, uint32_t* active,
                                          const float* origin3, float voxel_size, int X, int Y, int Z,
                                          const float* depth_f32, int num_frames, int img_h, int img_w,
                                          const float* frame_params, const dt_tsdf_thresholds* th, dt_stream_t s);
/* Voxel-slab form for multi-GPU fusion of large final volumes (alternative): the same update
 * restricted to the x-slab [x_begin, x_begin + x_count) of the FULL volume the pointers address -- voxel centres are
 * computed from the global index, so a volume assembled from the slabs of several ranks is bit-identical to one
 * integrated whole (tools/tsdf.py:414-558 per voxel).  depth: fp16 or (depth_is_f32) fp32 maps, as above. */
int dt_tsdf_integrate_frames_xslab_f16(uint16_t* values, uint16_t* weights, uint32_t* active,
                                       const float* origin3, float voxel_size, int X, int Y, int Z,
                                       int x_begin, int x_count, const void* depth, int depth_is_f32,
                                       int num_frames, int img_h, int img_w, const float* frame_params,
                                       const dt_tsdf_thresholds* th, dt_stream_t s);
/* replaces: TSDF.sample_tsdf (tools/tsdf.py:277-339), trilinear, align_corners=True, zeros
 * padding.  fp16_math = 0 reproduces the reference's CPU branch (fp32 math on the half volume,
 * pinned by goldens); 1 rounds grid and result to half like its GPU branch (unpinned).
 * origin3: HOST pointer (the half-rounded origin the reference keeps, as fp32). */
int dt_tsdf_sample_f16(const uint16_t* volume, const float* origin3, float voxel_size,
                       int X, int Y, int Z, const float* points_n3, float* out_n,
                       int64_t n, int fp16_math, dt_stream_t s);

/* ---- marching cubes over the active-voxel set -------------------------------------------
 * replaces: marching_cubes_(vol, isolevel, active_voxels, min_bounds, max_bounds)
 * (tools/marching_cubes/ext.cpp:4-6, marching_cubes.h:47-69, marching_cubes.cu:455-597)
 * with the CUDA path's semantics (active set, bounds, "corner < -0.99999 => skip").
 * Two-phase: dt_mc_count leaves per-block offsets in `workspace` and writes
 * counts_out[0] = cells, counts_out[1] = vertices (device ints; -1 on int overflow); the caller
 * reads them once, allocates verts [V,3] f32 / faces [V/3,3] i64 / ids [V] i64 and calls
 * dt_mc_generate with the same arguments.  min_bounds3 / max_bounds3: HOST int[3] in (i,j,k)
 * order or NULL.  Output vertex coordinates use the reference's (x,y,z) = (k,j,i) order.
 * Requirements checked by every entry point (error status otherwise): X*Y*Z is a multiple of 256
 * (TSDF dims are multiples of VOX_MOD=8) and `active` -- 1 bit per voxel, voxel v = bit v%32 of
 * word v/32 -- is 16-byte aligned (a workgroup reads its eight words as two 16-byte vectors).
 */
int64_t dt_mc_workspace_bytes(int X, int Y, int Z);
int dt_mc_count(const uint16_t* values_f16, const uint32_t* active, int X, int Y, int Z,
                float isolevel, const int* min_bounds3, const int* max_bounds3,
                void* workspace, int* counts_out, dt_stream_t s);
int dt_mc_generate(const uint16_t* values_f16, const uint32_t* active, int X, int Y, int Z,
                   float isolevel, const int* min_bounds3, const int* max_bounds3,
                   const void* workspace, float* verts_v3, int64_t* faces_f3, int64_t* ids_v,
                   int num_verts, dt_stream_t s);

/* ---- hint-mesh depth render --------------------------------------------
 * replaces: PyTorch3DMeshDepthRenderer.render (utils/rendering_utils.py:22-53) = PyTorch3D
 * MeshRasterizer(image_size=(h,w), blur_radius=0, faces_per_pixel=1).zbuf, background -1.
 * verts in world coordinates, faces int64 [F,3]; cam_T_world_44 / K_44 (PIXEL-unit intrinsics):
 * device, 16 floats row-major; workspace_hw: h*w uint32.  Parity with PyTorch3D is unpinned. */
int dt_raster_depth_f32(const float* verts_v3, const int64_t* faces_f3, int64_t num_faces,
                        const float* cam_T_world_44, const float* K_44, int h, int w,
                        uint32_t* workspace_hw, float* depth_hw, dt_stream_t s);
/* The same render for the raw triangle soup of dt_mc_generate (vertex 3f+i of face f, (k,j,i) voxel-index
 * coordinates; world = origin + (i,j,k)*voxel_size): skips the id sort/unique vertex merge of
 * utils/pytorch3d_extras.py:90-106, which a depth render does not need.  origin3: HOST pointer. */
int dt_raster_soup_depth_f32(const float* verts_kji_v3, int64_t num_faces, const float* origin3,
                             float voxel_size, const float* cam_T_world_44, const float* K_44, int h, int w,
                             uint32_t* workspace_hw, float* depth_hw, dt_stream_t s);
/* Marching cubes and the depth render of its surface in ONE pass, for the per-frame hint of the incremental mode
 * (test_incremental.py:204-258: tsdf.to_mesh_pytorch3d + PyTorch3DMeshDepthRenderer.render): every workgroup
 * compacts the triangles of its 256 cells in LDS and rasterises them straight into the z-buffer.  No vertex buffer
 * and no vertex count on the host (dt_mc_count's one host read per frame); depth_hw is bit-identical to
 * dt_mc_count + dt_mc_generate + dt_raster_soup_depth_f32.  Arguments as in those calls. */
int dt_mc_raster_depth_f32(const uint16_t* values_f16, const uint32_t* active, int X, int Y, int Z,
                           float isolevel, const int* min_bounds3, const int* max_bounds3,
                           const float* origin3, float voxel_size, const float* cam_T_world_44,
                           const float* K_44, int h, int w, uint32_t* workspace_hw, float* depth_hw,
                           dt_stream_t s);
/* Hint maps from a rendered depth in one pass (test_incremental.py:204-258): back-project pixel centres
 * with invK / world_T_cam (device, 16 floats each, row-major 4x4), trilinearly sample the fused
 * weight volume, keep depth where rendered (!= -1) and weight >= threshold.  Outputs [h,w]:
 * hint (NaN where dropped), mask (1/0 float), mask_b (1/0 bytes), sampled weights (0 where dropped).
 * fp16_math: as in dt_tsdf_sample_f16 (0 = fp32 blend on the half volume, the pinned branch; 1 = grid, result and cut in
 * half like the reference's device branch, unpinned). */
int dt_hint_from_depth_f32(const float* depth_hw, const uint16_t* weights_vol_f16, const float* origin3,
                           float voxel_size, int X, int Y, int Z, const float* invK_44,
                           const float* world_T_cam_44, float threshold, int h, int w,
                           float* hint_hw, float* mask_hw, uint8_t* mask_b_hw,
                           float* sampled_weights_hw, int fp16_math, dt_stream_t s);

/* ---- voxel-block (sparse) fp32 TSDF ------------------------------------------
 * replaces: CustomOpen3dFuser (tools/fusers_helper.py:263-511) over Open3D's VoxelBlockGrid (open3d==0.18.0,
 * third party: algorithm restated, parity unpinned).  The grid is seven caller-owned device buffers:
 *   dir      int32 [nb^3]      block directory over block coordinates [-nb/2, nb/2)^3, -1 = unallocated (init -1)
 *   touch    uint8 [nb^3]      per-frame marks (init 0)
 *   keys     int32 [cap*3]     block coordinates per slot
 *   tsdf, weight fp32 [cap*4096]  16^3-voxel tiles, index (lx*16 + ly)*16 + lz (init 0)
 *   count2   int32 [2]         [0] allocated slots, [1] blocks that could not be placed (capacity / directory extent)
 * dt_sparse_integrate_f32 = compute_unique_block_coordinates + activate (:326-336) + update_tsdf_for_voxels (:369-441)
 * for ONE depth map [h,w] fp32 (device); K44 / cam_T_world44 are HOST pointers (16 floats, row-major).
 * trunc_voxels: truncation distance in voxels (reference: 3). */
int dt_sparse_block_voxels(void);
int dt_sparse_integrate_f32(int* dir, unsigned char* touch, int nb, float voxel_size, int* keys, float* tsdf, float* weight,
                            int* count2, int capacity, const float* depth_hw, int img_h, int img_w, const float* K44_host,
                            const float* cam_T_world44_host, float max_depth, float trunc_voxels, int extended_neg_truncation,
                            dt_stream_t s);
/* The same for num_frames depth maps [n,h,w] with their cameras in DEVICE memory ([n,16] floats each, row-major 4x4),
 * integrated in order: no host read of the cameras, hence no device synchronisation in the fusion loop
 * (tools/fusers_helper.py:288-336 loops over the batch on the host with .cpu() cameras). */
int dt_sparse_integrate_frames_f32(int* dir, unsigned char* touch, int nb, float voxel_size, int* keys, float* tsdf, float* weight,
                                   int* count2, int capacity, const float* depth_nhw, int num_frames, int img_h, int img_w,
                                   const float* K_n44_dev, const float* cam_T_world_n44_dev, float max_depth,
                                   float trunc_voxels, int extended_neg_truncation, dt_stream_t s);
/* trilinear sample of the tsdf (what=0) or weight (what=1) field at world points; unallocated corners read 0 */
int dt_sparse_sample_f32(int* dir, unsigned char* touch, int nb, float voxel_size, int* keys, float* tsdf, float* weight,
                         int* count2, int capacity, const float* points_N3, float* out_N, int64_t n, int what, dt_stream_t s);
/* replaces: VoxelBlockGrid.extract_triangle_mesh(weight_threshold) (:451-481): marching cubes over the first num_slots
 * slots; a cell is meshed when all 8 corners are allocated with weight > weight_threshold.  Two phases like dt_mc_*:
 * count fills slot_offsets[num_slots] (exclusive scan) and total_out[0] = vertex count; generate writes world-space
 * vertices [V,3], per-vertex interpolated weights [V] (may be NULL), faces [V/3,3] and int64 edge ids [V]. */
int dt_sparse_mc_count(int* dir, unsigned char* touch, int nb, float voxel_size, int* keys, float* tsdf, float* weight, int* count2,
                       int capacity, int num_slots, float isolevel, float weight_threshold, int* slot_offsets, int* total_out,
                       dt_stream_t s);
int dt_sparse_mc_generate(int* dir, unsigned char* touch, int nb, float voxel_size, int* keys, float* tsdf, float* weight,
                          int* count2, int capacity, int num_slots, float isolevel, float weight_threshold, const int* slot_offsets,
                          float* verts_v3, float* vert_weights_v, int64_t* faces_f3, int64_t* ids_v, int num_verts, dt_stream_t s);

/* ---- Winograd F(4x4, 3x3): the chip-filling 3x3 stride-1 layers with 2.25 multiplies per output pixel (csrc/conv_wino4.hip) ---
 * replaces: the same reference convolutions as dt_conv2d_wino_f32 (modules/layers.py:77-94 BasicBlock convs,
 * modules/networks_fast.py:17-40 ConvBlock convs, modules/networks.py:20-85 UNet++ nodes) -- same descriptor, same fused
 * concat / nearest-x2 / padding / bias / residual / activation semantics, exact-fp32 MFMA.  Output blocks are 16 x 16 pixels x
 * 32 channels (384-thread workgroups): meant for launches with enough blocks to fill the chip (dt_conv2d_wino4_blocks; the
 * host side picks F(2x2) below its threshold).  fp32 rounding is amplified more than by F(2x2) (about 5e-6 mean, 3e-5 worst per
 * layer on O(1) activations): inside the path's tolerances, checked by the whole-tensor parity tests.
 *   dt_conv_wino4_pack_floats(c_out, c_in)   floats of the packed weights (c_out * c_in * 36), 0 for unsupported channel counts
 *   dt_conv_wino4_pack_f32                   OIHW 3x3 -> U = G g G^T (computed in double, rounded once), packed for the kernel
 *   dt_conv2d_wino4_blocks(desc)             workgroups the launch would have; 0 = shape not supported
 *   dt_conv2d_wino4_f32                      the convolution; `packed_w` from dt_conv_wino4_pack_f32 */
int64_t dt_conv_wino4_pack_floats(int c_out, int c_in);
int dt_conv_wino4_pack_f32(const float* W_oihw, float* packed, int c_out, int c_in, dt_stream_t s);
int64_t dt_conv2d_wino4_blocks(const dt_conv_desc* d);
int dt_conv2d_wino4_f32(const dt_conv_desc* d, const float* in0, const float* in1, const float* in2, const float* packed_w,
                        const float* bias, const float* residual, float* out, dt_stream_t s);

/* ---- launch programs: one host call per model step ------------------------------------------------------------------
 * replaces: nothing the reference has as a function -- it is the host side of the call sequence of
 * DepthModelCVHint.forward (experiment_modules/doubletake_model.py:341-349,375-423: cost volume -> CVEncoder -> depth
 * decoder -> exp), which the reference enqueues op by op from Python.  Here the ~50 kernel launches of that sequence are
 * recorded once while they run through the entry points above, and re-issued by dt_program_launch as plain
 * hipLaunchKernel calls (no planning, no argument marshalling, no host-language call per launch).
 *
 *   dt_program_begin(s)        the calling THREAD starts recording the launches this library makes on stream s (they still
 *                              execute; launches on other streams are neither recorded nor disturbed)
 *   dt_program_input(p, n)     declares a device range [p, p+n) whose address differs between replays (an input tensor of the
 *                              step); ranges must not overlap; returns the slot index (>= 0) or -1
 *   dt_program_mark()          segment boundary at the current position; returns the index of the segment that starts here
 *                              (segment 0 starts at dt_program_begin) or -1
 *   dt_program_end(&prog)      stops recording; every POINTER of the recorded arguments that points into an input range becomes a
 *                              patch (slot, offset).  Pointers are known by position (pointer parameters; the pointer members
 *                              every by-value argument struct declares, csrc/common.hpp DT_ARG_POINTERS) -- never guessed from
 *                              the argument bytes, whose struct padding is uninitialised
 *   dt_program_abort()         stops recording and discards what was recorded (error paths)
 *   dt_program_launch(prog, segment, inputs, num_inputs, s)
 *                              re-issues the launches of one segment (segment = -1: all of them) on s, which must be the
 *                              stream the program was recorded on (the library's per-stream split-K scratch is baked in).
 *                              inputs[i] = this replay's address of slot i (same extents and layout as recorded); they are
 *                              applied when segment <= 0, i.e. once per replay.  One replay at a time per program.
 *   dt_program_info(prog, what) 0 launches, 1 segments, 2 patches, 3 input slots, 4 argument bytes, 5 argument words that are not
 *                              pointers but happen to hold a value inside an input range (diagnostic: never patched); -1 on error
 *   dt_program_free(prog)
 *
 * Everything else the recorded launches point at (intermediates, outputs, packed weights) must stay allocated, at the same
 * addresses, until dt_program_free; process-wide settings that pick kernels or grids (dt_conv_set_plan_objective,
 * dt_cv_mlp_set_cu_budget) are baked in at recording time. */
typedef void* dt_program_t;
int dt_program_begin(dt_stream_t s);
int dt_program_input(const void* base, int64_t bytes);
int dt_program_mark(void);
int dt_program_end(dt_program_t* prog_out);
int dt_program_abort(void);
int dt_program_launch(dt_program_t prog, int segment, const void* const* inputs, int num_inputs, dt_stream_t s);
int64_t dt_program_info(dt_program_t prog, int what);
int dt_program_free(dt_program_t prog);

#ifdef __cplusplus
}
#endif
#endif /* DOUBLETAKE_HIP_H */
