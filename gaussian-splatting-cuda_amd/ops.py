"""The gsplat operator surface (gsplat/Ops.h:12-43,69-166 of the reference) on the HIP backend.

Everything here is the C++ shim `_gsx_ops` (csrc/ops_shim.cpp) over the C ABI of libgsx.so.  There is NO
fallback: if the native module is missing or cannot be loaded this import fails loudly.
"""
import os
import sys

import torch  # noqa: F401  (loads libamdhip64 / libtorch before the extension)

_HERE = os.path.dirname(os.path.abspath(__file__))
if _HERE not in sys.path:
    sys.path.insert(0, _HERE)
try:
    import _gsx_ops as _C
except ImportError as e:  # pragma: no cover
    raise ImportError(
        "gsx: the native HIP extension (_gsx_ops / libgsx.so) is not built or failed to load; run "
        "`python __graft_entry__.py` (build()) first. There is no CPU or PyTorch fallback. Cause: %s" % e)

CameraModelType = _C.CameraModelType
ShutterType = _C.ShutterType
UnscentedTransformParameters = _C.UnscentedTransformParameters

spherical_harmonics_fwd = _C.spherical_harmonics_fwd
spherical_harmonics_bwd = _C.spherical_harmonics_bwd
intersect_tile = _C.intersect_tile
intersect_offset = _C.intersect_offset
projection_ut_3dgs_fused = _C.projection_ut_3dgs_fused


def rasterize_to_pixels_from_world_3dgs_fwd(*args, keep_ws=False):
    """gsplat::rasterize_to_pixels_from_world_3dgs_fwd; keep_ws=True also returns the workspace (packed per-Gaussian records)
    that the backward of the same inputs can take back (fwd_ws=) instead of re-packing."""
    return _C.rasterize_fwd_keep_ws(*args) if keep_ws else _C.rasterize_to_pixels_from_world_3dgs_fwd(*args)


def rasterize_to_pixels_from_world_3dgs_bwd(*args, fwd_ws=None, lists=None):
    """`lists`: the IsectLists handle of intersect_tile_binned_guarded the forward ran with (guarded protocol, include/gsx.h)."""
    return _C.rasterize_to_pixels_from_world_3dgs_bwd(*args, fwd_ws, lists)


def rasterize_bwd_act(*args, fwd_ws=None, lists=None, raw=None, out=(None, None, None), reg=(0.0, 0.0)):
    """The blend backward of ONE camera through to the raw SplatData parameters (include/gsx.h, ABI 7): `args` as for
    rasterize_to_pixels_from_world_3dgs_bwd, raw = (scaling_raw, rotation_raw, opacity_raw [N]), out = optional gradient buffers, reg = the
    regulariser gradients per element.  Returns (v_means, v_colors, v_scaling_raw, v_rotation_raw, v_opacity_raw)."""
    return _C.rasterize_bwd_act(*args, fwd_ws, lists, raw[0], raw[1], raw[2], out[0], out[1], out[2], float(reg[0]), float(reg[1]))


quats_to_rotmats = _C.quats_to_rotmats
relocation = _C.relocation
add_noise = _C.add_noise
abi_version = _C.abi_version

# fused glue ops (extensions beyond Ops.h; include/gsx.h "fused glue")
sh_colors_fwd = _C.sh_colors_fwd
sh_colors_bwd = _C.sh_colors_bwd
sh_colors_bwd_adam = _C.sh_colors_bwd_adam
splat_activations_fwd = _C.splat_activations_fwd
splat_activations_projection_ut = _C.splat_activations_projection_ut
frontend_fused_render = _C.frontend_fused_render   # the same launch without the conics output (rasterize_fused)
frontend_fused = _C.frontend_fused            # activations -> UT projection -> SH colours -> packed records, one kernel (gsx_frontend.hip)
rasterize_fwd_packed = _C.rasterize_fwd_packed
splat_activations_bwd = _C.splat_activations_bwd
adam_step = _C.adam_step
adam_step_multi = _C.adam_step_multi
adam_step_wrapper = _C.adam_step_wrapper


# The optimizer operators over many tensors (include/gsx_optim.h).  Any number of tensors in a list, empty ones included; float32, bfloat16 or float16
# parameters and gradients, dense or row-strided views (sh[:, 1:]); everything on one device, on its current stream; nothing waits for the device, all of them
# may be captured into a graph (the numbers of the call are captured with it; step, clip factor and skip flag come from the control block).
MOMENT_RUN = _C.MOMENT_RUN   # consecutive values of a tensor that share a scale of the 8-bit moments


def step_control(device, step=0):
    """The block through which grad_norm_multi steers the updates behind it without the host: float64 [norm, factor, skip, step, 4 internal words].  One block for
    each sequence of calls (two streams, or two graphs in flight at once, take one each)."""
    c = torch.zeros(_C.CONTROL_WORDS, dtype=torch.float64, device=device)
    c[1], c[3] = 1.0, float(step)
    return c


def grad_norm_multi(grads, control, max_norm=float("inf")):
    """control[0] = the norm of all gradients (accumulated in 64 bits, the same bits every time), [1] = min(1, max_norm / (norm + 1e-6)), [2] = 1 if a gradient
    is infinite or NaN ([1] is 0 then, and the updates that read the block leave everything as it is), [3] (the step) advanced by one if none is."""
    _C.grad_norm_multi(grads, control, max_norm)


def adamw_step_multi(params, exp_avgs, exp_avg_sqs, grads, lrs, weight_decays, beta1, beta2, eps, steps, control=None, splits=()):
    """AdamW with decoupled decay on every tensor of the lists, in place: moments contiguous float32, a rate and a decay for each tensor.  16-bit parameters are rounded to
    nearest after the step (a step below half a place of theirs leaves them where they are).  No two tensors of the lists may share memory.  The parameters' version
    counters advance: a backward through a graph from before the step that needs their old values is refused, as behind the library's own optimizers.
    steps: the number of this step for each tensor, from 1; empty: the control block's.  control (step_control): the gradients are multiplied by its factor,
    and nothing is changed where its skip flag is set.  splits, one for each tensor or empty: (split, lr_b, weight_decay_b, hold_a, hold_b) — the columns
    [split, ...) of a tensor seen as rows are a second group with its own rate and decay (0: one group); a held group and its moments stay as they are."""
    _C.adamw_step_multi(params, exp_avgs, exp_avg_sqs, grads, lrs, weight_decays, beta1, beta2, eps, steps, control, splits)


def adamw8_step_multi(params, exp_avgs, exp_rmss, avg_scales, rms_scales, grads, lrs, weight_decays, beta1, beta2, eps, steps, control=None, splits=(), seed=None):
    """adamw_step_multi with the first moment and the root of the second as float8_e4m3fn tensors, each with one float32 scale for MOMENT_RUN consecutive values
    (float32 [ceil(numel / MOMENT_RUN)]; zeros are zero moments).  seed None: rounded to nearest; 0 .. 2^32 - 1: stochastically, another draw for
    every step, tensor of the list and value.  A held group's parameters stay as they are, its moments as values: they are rounded anew with their run, whose scale the
    other group may move.  With rounding to nearest a moment that changes by less than half a step of the format (3 to 6 %) does not
    change at all, and the second moment's average over 1 / (1 - beta2) steps comes to rest: training takes a seed."""
    _C.adamw8_step_multi(params, exp_avgs, exp_rmss, avg_scales, rms_scales, grads, lrs, weight_decays, beta1, beta2, eps, steps, control, splits, seed)


def adamw8_select_rows(exp_avgs, exp_rmss, avg_scales, rms_scales, index):
    """Rows of 8-bit moments (permuted, removed, repeated, added) as new tensors: row j is row index[j] of the old ones, zero where index[j] is outside them.
    All tensors have the same number of rows.  Returns the four lists."""
    return _C.adamw8_select_rows(exp_avgs, exp_rmss, avg_scales, rms_scales, index)


intersect_tile_binned = _C.intersect_tile_binned
intersect_tile_binned_guarded = _C.intersect_tile_binned_guarded   # no host read of n_isects: (tiles_per_gauss, flatten_ids [capacity], offsets, IsectLists)
shim_guarded_stats = _C.shim_guarded_stats
intersect_tile_device_sort = _C.intersect_tile_device_sort
adam_step_split = _C.adam_step_split
fusedssim = _C.fusedssim
fusedssim_backward = _C.fusedssim_backward
photometric_loss_fwd = _C.photometric_loss_fwd
photometric_loss_bwd = _C.photometric_loss_bwd
photometric_loss_single_pass = _C.photometric_loss_single_pass   # loss3 and v_render in one kernel (include/gsx.h ABI 7)
shim_stats = _C.shim_stats
shim_ranked_calls = _C.shim_ranked_calls
