"""The extension-op boundary of the mapped-convolution backend.

Same op names, argument order and return values as the reference's pybind
modules under `_mapped_convolution_ext` (one module per op family there, one
namespace here); each function checks its tensors like the reference's
include/nn/layers/*.h wrappers do, allocates the outputs with torch, and calls
the C ABI of libmcx_hip.so on the current HIP stream.  Tensors must live on the
GPU: there is no CPU implementation behind these names.
"""
import array
import contextlib

import torch

from . import _lib
from ._lib import MCX_BF16, MCX_F32, MCX_F64

_DTYPES = {torch.float32: MCX_F32, torch.float64: MCX_F64, torch.bfloat16: MCX_BF16}


# Optional timing hook: when set to a list, every C-ABI call made by the convolution
# ops appends (label, start_event, end_event), recorded on the stream the kernels
# are enqueued on.  Used by the benchmark to time individual kernels.
profile_events = None
profile_pool = []  # pre-made (start, end) event pairs, see make_event_pool

# resample_to_map and the unpoolings run as gathers through a transposed map when
# given a workspace; False selects the library's atomic-scatter form instead.
scatter_as_gather = True


def make_event_pool(n, device):
    """n pairs of timing events whose underlying handles exist (an event gets its handle at
    its first record), for `profile_pool`."""
    stream = torch.cuda.current_stream(device)
    pool = []
    for _ in range(n):
        pair = (torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True))
        for e in pair:
            e.record(stream)
        pool.append(pair)
    return pool


def _timed(label, device, fn):
    """Run one C-ABI call; with `profile_events` set and a pair left in `profile_pool`, ask
    the library to record the pair around the call's dominant kernel (the only cost inside
    a timed region: one extra C call and two event records)."""
    if profile_events is None or not profile_pool:
        return fn()
    start, end = profile_pool.pop()
    lib = _lib.load()
    lib.mcx_profile_dominant_kernel(start.cuda_event, end.cuda_event)
    rc = fn()
    lib.mcx_profile_dominant_kernel(None, None)
    profile_events.append((label, start, end))
    return rc


def _contig(**tensors):
    for name, t in tensors.items():
        if t is not None and not t.is_contiguous():
            raise RuntimeError("%s must be contiguous" % name)


def _on_gpu(ref_name, ref, **tensors):
    if not ref.is_cuda:
        raise RuntimeError(
            "%s must be a GPU tensor: this backend has no CPU implementation" % ref_name)
    device = ref.get_device()
    for name, t in tensors.items():
        if t is not None and t.get_device() != device:
            raise RuntimeError("%s must be on the same device as %s" % (name, ref_name))


def _dtype(data, maps=(), same=()):
    """Data dtype code.  Maps share the data's dtype (the reference's rule,
    layers/nn/layer_utils.py:21-30), except bf16 data which takes fp32 maps
    because bf16 cannot hold pixel coordinates above 256 exactly."""
    if data.dtype not in _DTYPES:
        raise RuntimeError("unsupported dtype %s" % data.dtype)
    want_map = torch.float32 if data.dtype == torch.bfloat16 else data.dtype
    for m in maps:
        if m is not None and m.dtype != want_map:
            raise RuntimeError("sample_map / interp_weights must be %s for %s data (got %s)" %
                               (want_map, data.dtype, m.dtype))
    for t in same:
        if t is not None and t.dtype != data.dtype:
            raise RuntimeError("tensor dtypes differ: %s vs %s" % (t.dtype, data.dtype))
    return _DTYPES[data.dtype]


def _ptr(t):
    return None if t is None else t.data_ptr()


# (the handle alone: a Stream object takes two microseconds to make, a call of a small layer thirty)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(t):
    if _raw_stream is None:
        return torch.cuda.current_stream(t.device).cuda_stream
    return _raw_stream(t.get_device())


def _changed(tensors):
    """Tells torch which tensors a kernel has written in place: graphs that have saved them refuse their
    backward pass then, and plans of a map are made anew."""
    torch.autograd.graph.increment_version(tensors)


_here = contextlib.nullcontext()


def _device(t):
    """A context in which t's device is the current one: nothing to switch where it is already."""
    return _here if torch.cuda.current_device() == t.get_device() else torch.cuda.device(t.device)


def _workspace(nbytes, device):
    """Scratch for one call (torch's caching allocator returns 512-byte aligned blocks)."""
    return torch.empty((max(int(nbytes), 1),), dtype=torch.uint8, device=device)


def _conv_workspace(nbytes, dt, device):
    """Scratch of a convolution call and its size.  float64 data needs none (the library then runs
    its scalar kernels), so a call that leaves no memory for it goes through without."""
    try:
        return _workspace(nbytes, device), nbytes
    except torch.OutOfMemoryError:
        if dt != MCX_F64:
            raise
        return None, 0


def _weighted_dims(sample_map, interp_weights, kernel):
    """Number of interpolation points P (0 = unweighted) after a shape check."""
    want = (4 if kernel else 3) + (0 if interp_weights is None else 1)
    if sample_map.dim() != want or sample_map.shape[-1] != 2:
        raise RuntimeError("sample_map has shape %s, expected %d dims ending in 2" %
                           (tuple(sample_map.shape), want))
    if interp_weights is None:
        return 0
    if tuple(interp_weights.shape) != tuple(sample_map.shape[:-1]):
        raise RuntimeError("interp_weights shape %s does not match sample_map %s" %
                           (tuple(interp_weights.shape), tuple(sample_map.shape)))
    return int(interp_weights.shape[-1])


# --------------------------------------------------------------------------- conv
def _conv_forward(input, sample_map, interp_weights, weight, bias, kernel_size, interpolation,
                  plan=None):
    _contig(input=input, sample_map=sample_map, interp_weights=interp_weights, weight=weight,
            bias=bias)
    _on_gpu("input", input, sample_map=sample_map, interp_weights=interp_weights, weight=weight,
            bias=bias)
    dt = _dtype(input, maps=(sample_map, interp_weights), same=(weight, bias))
    P = _weighted_dims(sample_map, interp_weights, True)
    B, Ci, IH, IW = input.shape
    Co = weight.shape[0]
    OH, OW, K = sample_map.shape[0], sample_map.shape[1], int(kernel_size)
    if weight.dim() != 3 or weight.shape[1] != Ci or weight.shape[2] != K or sample_map.shape[2] != K:
        raise RuntimeError("weight %s / sample_map %s do not match input channels %d, kernel %d" %
                           (tuple(weight.shape), tuple(sample_map.shape), Ci, K))
    if bias.numel() != Co:
        raise RuntimeError("bias must have %d elements" % Co)
    out = torch.empty((B, Co, OH, OW), dtype=input.dtype, device=input.device)
    lib = _lib.load()
    ws, ws_bytes = _conv_workspace(
        lib.mcx_conv_forward_workspace(B, Ci, Co, IH, IW, OH, OW, K, P, dt), dt, input.device)
    if plan is None and map_plan_cache is not None:
        plan = _cached_plan(sample_map, interp_weights, IH, IW, interpolation, input.dtype)
    plan_ptr, plan_bytes, plan_desc = _plan_args(plan)
    with _device(input):
        rc = _timed("conv_forward", input.device, lambda: lib.mcx_conv_forward_planned(
            _ptr(input), _ptr(sample_map), _ptr(interp_weights), _ptr(weight), _ptr(bias),
            _ptr(out), _ptr(ws), ws_bytes, plan_ptr, plan_bytes, plan_desc, B, Ci, Co, IH, IW, OH,
            OW, K, P, int(interpolation), dt, _stream(input)))
    _lib.check(rc, "mapped_conv_forward")
    return out


# ---- map plans (no counterpart in the reference) ------------------------------------
# What the operators derive from sample_map alone can be built once and reused while the map
# does not change: for the (transposed) convolutions the transposed map of the scatter
# direction, the resolved taps of the gather direction and the masks of pairs in use
# (`conv_map_plan`); for resample_to_map and the unpoolings the sorted per-destination lists of
# contributions (`scatter_map_plan`).  With `map_plan_cache` set to a dict (see
# enable_map_plan_cache) the ops keep the plans of the maps they have seen, keyed by the
# tensors' storage and in-place version counters.  Off by default: every call then rebuilds
# what it needs, like the reference.
map_plan_cache = None
_MAP_PLAN_CACHE_ENTRIES = 16


class MapPlan:
    """A map plan: the device buffer, the host-side descriptor the library checks it by
    (mcx_plan_desc: op family, interpolation, sizes, the addresses of the plan and of the map it
    was built from) and the map tensors themselves, kept alive so that their addresses cannot
    pass to other tensors while the plan exists."""
    __slots__ = ("buffer", "desc", "tensors")

    def __init__(self, buffer, desc, tensors):
        self.buffer, self.desc, self.tensors = buffer, desc, tensors

    def numel(self):
        return self.buffer.numel()


def _plan_args(plan):
    """(device pointer, bytes, descriptor) of a MapPlan for the C ABI; NULLs for None."""
    if plan is None:
        return None, 0, None
    if not isinstance(plan, MapPlan):
        raise RuntimeError("plan must come from conv_map_plan / scatter_map_plan / pool_map_plan")
    import ctypes
    return plan.buffer.data_ptr(), plan.buffer.numel(), ctypes.byref(plan.desc)


def enable_map_plan_cache(enabled=True):
    """Keep (or stop keeping) the plans of the sample maps seen by the convolution backward."""
    global map_plan_cache
    map_plan_cache = {} if enabled else None


def conv_map_plan(sample_map, interp_weights, input_height, input_width, interpolation,
                  data_dtype=torch.float32):
    """Plan of one sample_map [MH, MW, K, (P,) 2] that samples an image of input_height x
    input_width: a MappedConvolution's input, or a MappedTransposedConvolution's OUTPUT.  None
    where the library has no plan for the case (float64 data, P > 4).  Pass it as `plan=` to
    the forward and backward ops of that layer for as long as the map's contents stay the
    same."""
    _contig(sample_map=sample_map, interp_weights=interp_weights)
    _on_gpu("sample_map", sample_map, interp_weights=interp_weights)
    P = _weighted_dims(sample_map, interp_weights, True)
    OH, OW, K = sample_map.shape[:3]
    dt = _DTYPES[data_dtype]
    want = torch.float32 if data_dtype == torch.bfloat16 else data_dtype
    if sample_map.dtype != want:
        raise RuntimeError("sample_map must be %s for %s data" % (want, data_dtype))
    lib = _lib.load()
    IH, IW = int(input_height), int(input_width)
    nbytes = lib.mcx_conv_plan_bytes(IH, IW, OH, OW, K, P, dt)
    if nbytes == 0:
        return None
    plan = torch.empty((nbytes,), dtype=torch.uint8, device=sample_map.device)
    desc = _lib.PlanDesc()
    with _device(sample_map):
        rc = lib.mcx_conv_plan_build(_ptr(sample_map), _ptr(interp_weights), _ptr(plan), nbytes,
                                     desc, IH, IW, OH, OW, K, P, int(interpolation), dt,
                                     _stream(sample_map))
    _lib.check(rc, "conv_map_plan")
    return MapPlan(plan, desc, (sample_map, interp_weights))


def _cached_plan(sample_map, interp_weights, IH, IW, interpolation, data_dtype, kind="conv",
                 **scatter_args):
    """Plan from the cache, rebuilt when a tensor was modified in place or replaced."""
    def ident(t):
        return None if t is None else (t.data_ptr(), t._version, tuple(t.shape))
    key = (kind, ident(sample_map), ident(interp_weights), IH, IW, int(interpolation), data_dtype,
           sample_map.device.index)
    hit = map_plan_cache.get(key)
    if hit is not None:
        return hit[0]
    if kind == "conv":
        plan = conv_map_plan(sample_map, interp_weights, IH, IW, interpolation, data_dtype)
    else:
        plan = scatter_map_plan(sample_map, interp_weights, IH, IW, interpolation,
                                for_max_unpool=kind == "max_unpool", **scatter_args)
    if len(map_plan_cache) >= _MAP_PLAN_CACHE_ENTRIES:
        map_plan_cache.pop(next(iter(map_plan_cache)))
    # the entry keeps the tensors alive, so their addresses cannot be handed to other maps
    map_plan_cache[key] = (plan, sample_map, interp_weights)
    return plan


def _conv_backward(grad_output, sample_map, interp_weights, input, weight, bias, kernel_size,
                   interpolation, plan=None, needs=(True, True, True)):
    _contig(input=input, sample_map=sample_map, interp_weights=interp_weights, weight=weight,
            bias=bias)
    grad_output = grad_output.contiguous()  # the reference reads it raw without a check
    _on_gpu("grad_output", grad_output, input=input, sample_map=sample_map,
            interp_weights=interp_weights, weight=weight, bias=bias)
    dt = _dtype(input, maps=(sample_map, interp_weights), same=(weight, grad_output))
    P = _weighted_dims(sample_map, interp_weights, True)
    B, Ci, IH, IW = input.shape
    Co, OH, OW = grad_output.shape[1], grad_output.shape[2], grad_output.shape[3]
    K = int(kernel_size)
    if tuple(weight.shape) != (Co, Ci, K) or tuple(sample_map.shape[:3]) != (OH, OW, K):
        raise RuntimeError("shape mismatch in mapped_conv_backward")
    # `needs` (grad_input, grad_weight, grad_bias): a gradient nobody asked for is not
    # computed (the C ABI takes NULL for it) and comes back as None
    grad_input = torch.empty_like(input) if needs[0] else None
    grad_weight = torch.empty_like(weight) if needs[1] else None
    grad_bias = torch.empty((Co,), dtype=input.dtype, device=input.device) if needs[2] else None
    lib = _lib.load()
    ws, ws_bytes = _conv_workspace(
        lib.mcx_conv_backward_workspace(B, Ci, Co, IH, IW, OH, OW, K, P, dt), dt, input.device)
    if plan is None and map_plan_cache is not None:
        plan = _cached_plan(sample_map, interp_weights, IH, IW, interpolation, input.dtype)
    plan_ptr, plan_bytes, plan_desc = _plan_args(plan)
    # Where kernels are timed, two C-ABI calls (NULL skips a gradient), so that the input gradient
    # and the weight gradient can be timed alone; the bias gradient rides on the weight
    # gradient's pass over grad_output.
    if profile_events is None:
        outs = {"conv_backward": (grad_input, grad_weight, grad_bias)}
    else:
        outs = {"conv_backward_input": (grad_input, None, None),
                "conv_backward_weight": (None, grad_weight, grad_bias)}
    with _device(input):
        for label, (gx, gw, gb) in outs.items():
            if gx is None and gw is None and gb is None:
                continue
            rc = _timed(label, input.device, lambda: lib.mcx_conv_backward_planned(
                _ptr(grad_output), _ptr(sample_map), _ptr(interp_weights), _ptr(input),
                _ptr(weight), _ptr(gx), _ptr(gw), _ptr(gb), _ptr(ws), ws_bytes, plan_ptr,
                plan_bytes, plan_desc, B, Ci, Co, IH, IW, OH, OW, K, P, int(interpolation), dt,
                _stream(input)))
            _lib.check(rc, "mapped_conv_backward")
    return [grad_input, grad_weight, grad_bias]


def mapped_conv_forward(input, sample_map, weight, bias, kernel_size, interpolation, plan=None):
    """include/nn/layers/mapped_convolution_layer.h:64-66.  `plan` (optional, not in the
    reference): see conv_map_plan."""
    return _conv_forward(input, sample_map, None, weight, bias, kernel_size, interpolation, plan)


def mapped_conv_backward(grad_output, sample_map, input, weight, bias, kernel_size, interpolation,
                         plan=None, needs=(True, True, True)):
    """include/nn/layers/mapped_convolution_layer.h:90-93 -> [grad_input, grad_weight, grad_bias].
    `plan` (optional, not in the reference): see conv_map_plan.  `needs` (optional, not in the
    reference): which of the three gradients to compute; the others come back as None."""
    return _conv_backward(grad_output, sample_map, None, input, weight, bias, kernel_size,
                          interpolation, plan, needs)


def weighted_mapped_conv_forward(input, sample_map, interp_weights, weight, bias, kernel_size,
                                 interpolation, plan=None):
    """include/nn/layers/weighted_mapped_convolution_layer.h:65-68.  `plan`: see conv_map_plan."""
    return _conv_forward(input, sample_map, interp_weights, weight, bias, kernel_size,
                         interpolation, plan)


def weighted_mapped_conv_backward(grad_output, sample_map, interp_weights, input, weight, bias,
                                  kernel_size, interpolation, plan=None,
                                  needs=(True, True, True)):
    """include/nn/layers/weighted_mapped_convolution_layer.h:97-100.  `plan`: see conv_map_plan;
    `needs`: see mapped_conv_backward."""
    return _conv_backward(grad_output, sample_map, interp_weights, input, weight, bias,
                          kernel_size, interpolation, plan, needs)


# ---------------------------------------------------------------- transposed conv
def _tconv_forward(input, sample_map, interp_weights, weight, bias, output_height, output_width,
                   kernel_size, interpolation, plan=None):
    _contig(input=input, sample_map=sample_map, interp_weights=interp_weights, weight=weight,
            bias=bias)
    _on_gpu("input", input, sample_map=sample_map, interp_weights=interp_weights, weight=weight,
            bias=bias)
    dt = _dtype(input, maps=(sample_map, interp_weights), same=(weight, bias))
    P = _weighted_dims(sample_map, interp_weights, True)
    B, Ci, IH, IW = input.shape
    Co, K = weight.shape[1], int(kernel_size)
    OH, OW = int(output_height), int(output_width)
    if tuple(weight.shape) != (Ci, Co, K) or tuple(sample_map.shape[:3]) != (IH, IW, K):
        raise RuntimeError("shape mismatch in mapped_transposed_conv_forward")
    out = torch.empty((B, Co, OH, OW), dtype=input.dtype, device=input.device)
    lib = _lib.load()
    ws, ws_bytes = _conv_workspace(
        lib.mcx_tconv_forward_workspace(B, Ci, Co, IH, IW, OH, OW, K, P, dt), dt, input.device)
    if plan is None and map_plan_cache is not None:
        plan = _cached_plan(sample_map, interp_weights, OH, OW, interpolation, input.dtype)
    plan_ptr, plan_bytes, plan_desc = _plan_args(plan)
    with _device(input):
        rc = lib.mcx_tconv_forward_planned(_ptr(input), _ptr(sample_map), _ptr(interp_weights),
                                           _ptr(weight), _ptr(bias), _ptr(out), _ptr(ws),
                                           ws_bytes, plan_ptr, plan_bytes, plan_desc, B, Ci, Co,
                                           IH, IW, OH, OW, K, P, int(interpolation), dt,
                                           _stream(input))
    _lib.check(rc, "mapped_transposed_conv_forward")
    return out


def _tconv_backward(grad_output, sample_map, interp_weights, input, weight, bias, kernel_size,
                    interpolation, plan=None, needs=(True, True, True)):
    _contig(input=input, sample_map=sample_map, interp_weights=interp_weights, weight=weight,
            bias=bias)
    grad_output = grad_output.contiguous()
    _on_gpu("grad_output", grad_output, input=input, sample_map=sample_map,
            interp_weights=interp_weights, weight=weight, bias=bias)
    dt = _dtype(input, maps=(sample_map, interp_weights), same=(weight, grad_output))
    P = _weighted_dims(sample_map, interp_weights, True)
    B, Ci, IH, IW = input.shape
    Co, OH, OW = grad_output.shape[1], grad_output.shape[2], grad_output.shape[3]
    K = int(kernel_size)
    if tuple(weight.shape) != (Ci, Co, K) or tuple(sample_map.shape[:3]) != (IH, IW, K):
        raise RuntimeError("shape mismatch in mapped_transposed_conv_backward")
    grad_input = torch.empty_like(input) if needs[0] else None
    grad_weight = torch.empty_like(weight) if needs[1] else None
    grad_bias = torch.empty((Co,), dtype=input.dtype, device=input.device) if needs[2] else None
    if not any(needs):
        return [None, None, None]
    lib = _lib.load()
    ws, ws_bytes = _conv_workspace(
        lib.mcx_tconv_backward_workspace(B, Ci, Co, IH, IW, OH, OW, K, P, dt), dt, input.device)
    if plan is None and map_plan_cache is not None:
        plan = _cached_plan(sample_map, interp_weights, OH, OW, interpolation, input.dtype)
    plan_ptr, plan_bytes, plan_desc = _plan_args(plan)
    with _device(input):
        rc = lib.mcx_tconv_backward_planned(
            _ptr(grad_output), _ptr(sample_map), _ptr(interp_weights), _ptr(input), _ptr(weight),
            _ptr(grad_input), _ptr(grad_weight), _ptr(grad_bias), _ptr(ws), ws_bytes, plan_ptr,
            plan_bytes, plan_desc, B, Ci, Co, IH, IW, OH, OW, K, P, int(interpolation), dt,
            _stream(input))
    _lib.check(rc, "mapped_transposed_conv_backward")
    return [grad_input, grad_weight, grad_bias]


def mapped_transposed_conv_forward(input, sample_map, weight, bias, output_height, output_width,
                                   kernel_size, interpolation, plan=None):
    """include/nn/layers/mapped_transposed_convolution_layer.h:64-69.  `plan` (optional, not in
    the reference): conv_map_plan(sample_map, None, output_height, output_width, ...)."""
    return _tconv_forward(input, sample_map, None, weight, bias, output_height, output_width,
                          kernel_size, interpolation, plan)


def mapped_transposed_conv_backward(grad_output, sample_map, input, weight, bias, kernel_size,
                                    interpolation, plan=None, needs=(True, True, True)):
    """include/nn/layers/mapped_transposed_convolution_layer.h:97-100.  `needs`: see
    mapped_conv_backward."""
    return _tconv_backward(grad_output, sample_map, None, input, weight, bias, kernel_size,
                           interpolation, plan, needs)


def weighted_mapped_transposed_conv_forward(input, sample_map, interp_weights, weight, bias,
                                            output_height, output_width, kernel_size,
                                            interpolation, plan=None):
    """include/nn/layers/weighted_mapped_transposed_convolution_layer.h:64-67."""
    return _tconv_forward(input, sample_map, interp_weights, weight, bias, output_height,
                          output_width, kernel_size, interpolation, plan)


def weighted_mapped_transposed_conv_backward(grad_output, sample_map, interp_weights, input,
                                             weight, bias, kernel_size, interpolation, plan=None,
                                             needs=(True, True, True)):
    """include/nn/layers/weighted_mapped_transposed_convolution_layer.h:98-100."""
    return _tconv_backward(grad_output, sample_map, interp_weights, input, weight, bias,
                           kernel_size, interpolation, plan, needs)


def scatter_map_plan(sample_map, interp_weights, dest_height, dest_width, interpolation,
                     for_max_unpool=False, kernel=None):
    """Plan of resample_to_map (sample_map [IH, IW, (P,) 2]) or of an unpooling (sample_map
    [OH, OW, K, (P,) 2]) into an image of dest_height x dest_width: the transposed form of the
    map, built once.  `kernel`: whether the map has a tap axis (default: told from its number of
    dimensions).  A plan built with `for_max_unpool` serves mapped_max_unpool only, one built
    without it resample_to_map / mapped_avg_unpool.  Pass it as `plan=` to those ops."""
    _contig(sample_map=sample_map, interp_weights=interp_weights)
    _on_gpu("sample_map", sample_map, interp_weights=interp_weights)
    if kernel is None:
        kernel = sample_map.dim() == (4 if interp_weights is None else 5)
    P = _weighted_dims(sample_map, interp_weights, kernel)
    if sample_map.dtype not in (torch.float32, torch.float64):
        raise RuntimeError("unsupported dtype %s" % sample_map.dtype)
    dt = _DTYPES[sample_map.dtype]
    MH, MW = sample_map.shape[0], sample_map.shape[1]
    K = sample_map.shape[2] if kernel else 1
    DH, DW = int(dest_height), int(dest_width)
    lib = _lib.load()
    nbytes = lib.mcx_scatter_plan_bytes(MH, MW, DH, DW, K, P, int(interpolation), dt)
    if nbytes == 0:
        return None
    plan = torch.empty((nbytes,), dtype=torch.uint8, device=sample_map.device)
    desc = _lib.PlanDesc()
    with _device(sample_map):
        rc = lib.mcx_scatter_plan_build(_ptr(sample_map), _ptr(interp_weights), _ptr(plan), nbytes,
                                        desc, MH, MW, DH, DW, K, P, int(interpolation), dt,
                                        1 if for_max_unpool else 0, _stream(sample_map))
    _lib.check(rc, "scatter_map_plan")
    return MapPlan(plan, desc, (sample_map, interp_weights))


def _scatter_plan_for(kind, plan, sample_map, interp_weights, DH, DW, interpolation, kernel):
    if plan is None and map_plan_cache is not None and scatter_as_gather:
        plan = _cached_plan(sample_map, interp_weights, DH, DW, interpolation, sample_map.dtype,
                            kind=kind, kernel=kernel)
    return plan


# ------------------------------------------------------------------------ pooling
def _pool_dims(input, sample_map, interp_weights, kernel_size):
    if input.dim() != 4:
        raise RuntimeError("expected a 4-D [B, C, H, W] tensor, got %d dimensions" % input.dim())
    P = _weighted_dims(sample_map, interp_weights, True)
    K = int(kernel_size)
    if sample_map.shape[2] != K:
        raise RuntimeError("sample_map kernel dimension %d != kernel_size %d" %
                           (sample_map.shape[2], K))
    return P, K


def _max_pool(input, sample_map, interp_weights, kernel_size, interpolation):
    _contig(input=input, sample_map=sample_map, interp_weights=interp_weights)
    _on_gpu("input", input, sample_map=sample_map, interp_weights=interp_weights)
    dt = _dtype(input, maps=(sample_map, interp_weights))
    P, K = _pool_dims(input, sample_map, interp_weights, kernel_size)
    B, C, IH, IW = input.shape
    OH, OW = sample_map.shape[0], sample_map.shape[1]
    out = torch.empty((B, C, OH, OW), dtype=input.dtype, device=input.device)
    idx = torch.empty((B, C, OH, OW), dtype=torch.int64, device=input.device)
    with _device(input):
        rc = _lib.load().mcx_max_pool(_ptr(input), _ptr(sample_map), _ptr(interp_weights),
                                      _ptr(out), _ptr(idx), B, C, IH, IW, OH, OW, K, P,
                                      int(interpolation), dt, _stream(input))
    _lib.check(rc, "mapped_max_pool")
    return [out, idx]


def _max_unpool(grad_output, idx_mask, sample_map, interp_weights, input_height, input_width,
                kernel_size, interpolation, plan=None):
    _contig(grad_output=grad_output, idx_mask=idx_mask, sample_map=sample_map,
            interp_weights=interp_weights)
    _on_gpu("grad_output", grad_output, idx_mask=idx_mask, sample_map=sample_map,
            interp_weights=interp_weights)
    dt = _dtype(grad_output, maps=(sample_map, interp_weights))
    if idx_mask.dtype != torch.int64 or idx_mask.shape != grad_output.shape:
        raise RuntimeError("idx_mask must be int64 with grad_output's shape")
    P, K = _pool_dims(grad_output, sample_map, interp_weights, kernel_size)
    B, C, OH, OW = grad_output.shape
    if tuple(sample_map.shape[:2]) != (OH, OW):
        raise RuntimeError("sample_map spatial size must match grad_output")
    IH, IW = int(input_height), int(input_width)
    gin = torch.empty((B, C, IH, IW), dtype=grad_output.dtype, device=grad_output.device)
    lib = _lib.load()
    plan = _scatter_plan_for("max_unpool", plan, sample_map, interp_weights, IH, IW,
                             interpolation, True)
    if plan is not None:
        with _device(grad_output):
            rc = lib.mcx_max_unpool_planned(_ptr(grad_output), _ptr(idx_mask), *_plan_args(plan),
                                            _ptr(gin), B, C, IH, IW, OH, OW, K, P,
                                            int(interpolation), dt, _stream(grad_output))
        _lib.check(rc, "mapped_max_unpool")
        return gin
    ws_bytes = lib.mcx_unpool_workspace(IH, IW, OH, OW, K, P, int(interpolation), dt) \
        if scatter_as_gather else 0
    ws = _workspace(ws_bytes, grad_output.device)
    with _device(grad_output):
        rc = lib.mcx_max_unpool(_ptr(grad_output), _ptr(idx_mask), _ptr(sample_map),
                                _ptr(interp_weights), _ptr(gin), _ptr(ws), ws_bytes, B, C, IH, IW,
                                OH, OW, K, P, int(interpolation), dt, _stream(grad_output))
    _lib.check(rc, "mapped_max_unpool")
    return gin


def _avg_pool(input, sample_map, interp_weights, kernel_size, interpolation):
    _contig(input=input, sample_map=sample_map, interp_weights=interp_weights)
    _on_gpu("input", input, sample_map=sample_map, interp_weights=interp_weights)
    dt = _dtype(input, maps=(sample_map, interp_weights))
    P, K = _pool_dims(input, sample_map, interp_weights, kernel_size)
    B, C, IH, IW = input.shape
    OH, OW = sample_map.shape[0], sample_map.shape[1]
    out = torch.empty((B, C, OH, OW), dtype=input.dtype, device=input.device)
    with _device(input):
        rc = _lib.load().mcx_avg_pool(_ptr(input), _ptr(sample_map), _ptr(interp_weights),
                                      _ptr(out), B, C, IH, IW, OH, OW, K, P, int(interpolation),
                                      dt, _stream(input))
    _lib.check(rc, "mapped_avg_pool")
    return out


def _avg_unpool(grad_output, sample_map, interp_weights, input_height, input_width, kernel_size,
                interpolation, plan=None):
    _contig(grad_output=grad_output, sample_map=sample_map, interp_weights=interp_weights)
    _on_gpu("grad_output", grad_output, sample_map=sample_map, interp_weights=interp_weights)
    dt = _dtype(grad_output, maps=(sample_map, interp_weights))
    P, K = _pool_dims(grad_output, sample_map, interp_weights, kernel_size)
    B, C, OH, OW = grad_output.shape
    if tuple(sample_map.shape[:2]) != (OH, OW):
        raise RuntimeError("sample_map spatial size must match grad_output")
    IH, IW = int(input_height), int(input_width)
    gin = torch.empty((B, C, IH, IW), dtype=grad_output.dtype, device=grad_output.device)
    lib = _lib.load()
    plan = _scatter_plan_for("avg_unpool", plan, sample_map, interp_weights, IH, IW,
                             interpolation, True)
    if plan is not None:
        with _device(grad_output):
            rc = lib.mcx_avg_unpool_planned(_ptr(grad_output), *_plan_args(plan), _ptr(gin),
                                            B, C, IH, IW, OH, OW, K, P, int(interpolation), dt,
                                            _stream(grad_output))
        _lib.check(rc, "mapped_avg_unpool")
        return gin
    ws_bytes = lib.mcx_unpool_workspace(IH, IW, OH, OW, K, P, int(interpolation), dt) \
        if scatter_as_gather else 0
    ws = _workspace(ws_bytes, grad_output.device)
    with _device(grad_output):
        rc = lib.mcx_avg_unpool(_ptr(grad_output), _ptr(sample_map), _ptr(interp_weights),
                                _ptr(gin), _ptr(ws), ws_bytes, B, C, IH, IW, OH, OW, K, P,
                                int(interpolation), dt, _stream(grad_output))
    _lib.check(rc, "mapped_avg_unpool")
    return gin


def mapped_max_pool(input, sample_map, kernel_size, interpolation):
    """include/nn/layers/mapped_max_pooling_layer.h:46-49 -> [pooled, idx_mask]."""
    return _max_pool(input, sample_map, None, kernel_size, interpolation)


def mapped_max_unpool(grad_output, idx_mask, sample_map, input_height, input_width, kernel_size,
                      interpolation, plan=None):
    """include/nn/layers/mapped_max_pooling_layer.h:69-73.  `plan`: see scatter_map_plan."""
    return _max_unpool(grad_output, idx_mask, sample_map, None, input_height, input_width,
                       kernel_size, interpolation, plan)


def weighted_mapped_max_pool(input, sample_map, interp_weights, kernel_size, interpolation):
    """include/nn/layers/weighted_mapped_max_pooling_layer.h:42-44."""
    return _max_pool(input, sample_map, interp_weights, kernel_size, interpolation)


def weighted_mapped_max_unpool(grad_output, idx_mask, sample_map, interp_weights, input_height,
                               input_width, kernel_size, interpolation, plan=None):
    """include/nn/layers/weighted_mapped_max_pooling_layer.h:67-70."""
    return _max_unpool(grad_output, idx_mask, sample_map, interp_weights, input_height,
                       input_width, kernel_size, interpolation, plan)


def mapped_avg_pool(input, sample_map, kernel_size, interpolation):
    """include/nn/layers/mapped_avg_pooling_layer.h:42-44."""
    return _avg_pool(input, sample_map, None, kernel_size, interpolation)


def mapped_avg_unpool(grad_output, sample_map, input_height, input_width, kernel_size,
                      interpolation, plan=None):
    """include/nn/layers/mapped_avg_pooling_layer.h:64-67.  `plan`: see scatter_map_plan."""
    return _avg_unpool(grad_output, sample_map, None, input_height, input_width, kernel_size,
                       interpolation, plan)


def weighted_mapped_avg_pool(input, sample_map, interp_weights, kernel_size, interpolation):
    """include/nn/layers/weighted_mapped_avg_pooling_layer.h:48-52."""
    return _avg_pool(input, sample_map, interp_weights, kernel_size, interpolation)


def weighted_mapped_avg_unpool(grad_output, sample_map, interp_weights, input_height, input_width,
                               kernel_size, interpolation, plan=None):
    """include/nn/layers/weighted_mapped_avg_pooling_layer.h:75-78."""
    return _avg_unpool(grad_output, sample_map, interp_weights, input_height, input_width,
                       kernel_size, interpolation, plan)


# ----------------------------------------------------------------------- resample
def _resample_to_map(input, sample_map, interp_weights, output_height, output_width,
                     interpolation, plan=None):
    _contig(input=input, sample_map=sample_map, interp_weights=interp_weights)
    _on_gpu("input", input, sample_map=sample_map, interp_weights=interp_weights)
    dt = _dtype(input, maps=(sample_map, interp_weights))
    P = _weighted_dims(sample_map, interp_weights, False)
    if input.dim() != 4:
        raise RuntimeError("expected a 4-D [B, C, H, W] tensor, got %d dimensions" % input.dim())
    B, C, IH, IW = input.shape
    if tuple(sample_map.shape[:2]) != (IH, IW):
        raise RuntimeError("sample_map spatial size must match the input")
    OH, OW = int(output_height), int(output_width)
    out = torch.empty((B, C, OH, OW), dtype=input.dtype, device=input.device)
    lib = _lib.load()
    plan = _scatter_plan_for("resample", plan, sample_map, interp_weights, OH, OW, interpolation,
                             False)
    if plan is not None:
        with _device(input):
            rc = lib.mcx_resample_to_map_planned(_ptr(input), *_plan_args(plan), _ptr(out),
                                                 B, C, IH, IW, OH, OW, P, int(interpolation), dt,
                                                 _stream(input))
        _lib.check(rc, "resample_to_map")
        return out
    ws_bytes = lib.mcx_resample_to_map_workspace(IH, IW, OH, OW, P, int(interpolation), dt) \
        if scatter_as_gather else 0
    ws = _workspace(ws_bytes, input.device)
    with _device(input):
        rc = lib.mcx_resample_to_map(_ptr(input), _ptr(sample_map), _ptr(interp_weights),
                                     _ptr(out), _ptr(ws), ws_bytes, B, C, IH, IW, OH, OW, P,
                                     int(interpolation), dt, _stream(input))
    _lib.check(rc, "resample_to_map")
    return out


def _resample_from_map(input, sample_map, interp_weights, interpolation):
    _contig(input=input, sample_map=sample_map, interp_weights=interp_weights)
    _on_gpu("input", input, sample_map=sample_map, interp_weights=interp_weights)
    dt = _dtype(input, maps=(sample_map, interp_weights))
    P = _weighted_dims(sample_map, interp_weights, False)
    if input.dim() != 4:
        raise RuntimeError("expected a 4-D [B, C, H, W] tensor, got %d dimensions" % input.dim())
    B, C, SH, SW = input.shape
    MH, MW = sample_map.shape[0], sample_map.shape[1]
    out = torch.empty((B, C, MH, MW), dtype=input.dtype, device=input.device)
    with _device(input):
        rc = _lib.load().mcx_resample_from_map(_ptr(input), _ptr(sample_map),
                                               _ptr(interp_weights), _ptr(out), B, C, SH, SW, MH,
                                               MW, P, int(interpolation), dt, _stream(input))
    _lib.check(rc, "resample_from_map")
    return out


def resample_to_map(input, sample_map, output_height, output_width, interpolation, plan=None):
    """include/nn/layers/resample_layer.h:38-40 (scatter).  `plan`: see scatter_map_plan."""
    return _resample_to_map(input, sample_map, None, output_height, output_width, interpolation,
                            plan)


def resample_from_map(input, sample_map, interpolation):
    """include/nn/layers/resample_layer.h:60-61 (gather)."""
    return _resample_from_map(input, sample_map, None, interpolation)


def weighted_resample_to_map(input, sample_map, interp_weights, output_height, output_width,
                             interpolation, plan=None):
    """include/nn/layers/weighted_resample_layer.h:49-54."""
    return _resample_to_map(input, sample_map, interp_weights, output_height, output_width,
                            interpolation, plan)


def weighted_resample_from_map(input, sample_map, interp_weights, interpolation):
    """include/nn/layers/weighted_resample_layer.h:78-81."""
    return _resample_from_map(input, sample_map, interp_weights, interpolation)


# ---------------------------------------------------------------------------- knn
def knn_forward(ref, query, k):
    """include/util/layers/knn_layer.h:25-35 -> [idx int64 [B,k,Q] (1-based), dist [B,k,Q]]."""
    _contig(ref=ref, query=query)
    _on_gpu("ref", ref, query=query)
    dt = _dtype(ref, same=(query,))
    if ref.dim() != 3 or query.dim() != 3 or ref.shape[:2] != query.shape[:2]:
        raise RuntimeError("ref and query must be [B, D, *] with equal B and D")
    B, D, R = ref.shape
    Q, k = query.shape[2], int(k)
    idx = torch.empty((B, k, Q), dtype=torch.int64, device=ref.device)
    dist = torch.empty((B, k, Q), dtype=ref.dtype, device=ref.device)
    lib = _lib.load()
    with _device(ref):
        # (the grid search's bins; 0 bytes where it does not apply and every point is walked)
        ws_bytes = lib.mcx_knn_workspace(B, D, R, dt)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=ref.device) if ws_bytes else None
        rc = lib.mcx_knn(_ptr(ref), _ptr(query), _ptr(idx), _ptr(dist),
                         _ptr(ws) if ws is not None else None, ws_bytes, B, D, R, Q, k, dt,
                         _stream(ref))
    _lib.check(rc, "knn_forward")
    return [idx, dist]


# ------------------------------------------------------- map builders, cube2rect
PROJECTIONS = {"grid": 0, "gnomonic": 1, "equirectangular": 2, "perspective": 3}


def projection_map(shape, kernel_size, proj, stride, dilation, device):
    """Sample map [ceil(H/stride), ceil(W/stride), kh*kw, 2] (float32, on `device`) of the
    reference's host-side builders, package/layers/util/spherical_projections.py:12-24,33-35;
    `proj` is a key of PROJECTIONS."""
    H, W = (int(v) for v in shape)
    kh, kw = (int(v) for v in kernel_size)
    stride, dilation = int(stride), int(dilation)
    device = torch.device(device)
    if device.type != "cuda":
        raise RuntimeError("maps are built on the GPU: this backend has no CPU implementation")
    out = torch.empty((-(-H // stride), -(-W // stride), kh * kw, 2), dtype=torch.float32,
                      device=device)
    with torch.cuda.device(device):
        rc = _lib.load().mcx_projection_map(_ptr(out), H, W, kh, kw, PROJECTIONS[proj], stride,
                                            dilation, _stream(out))
    _lib.check(rc, "projection_map")
    return out


def cube_projection_map(cube_dim, kernel_size, stride, device):
    """spherical_projections.py:26-30 -> [ceil(dim/stride), ceil(6*dim/stride), kh*kw, 2]."""
    dim, stride = int(cube_dim), int(stride)
    kh, kw = (int(v) for v in kernel_size)
    device = torch.device(device)
    if device.type != "cuda":
        raise RuntimeError("maps are built on the GPU: this backend has no CPU implementation")
    out = torch.empty((-(-dim // stride), -(-6 * dim // stride), kh * kw, 2),
                      dtype=torch.float32, device=device)
    with torch.cuda.device(device):
        rc = _lib.load().mcx_cube_projection_map(_ptr(out), dim, kh, kw, stride, _stream(out))
    _lib.check(rc, "cube_projection_map")
    return out


def cube2rect(cubemap, rect_height, rect_width, interpolation):
    """include/util/layers/cube2rect_layer.h:29-43: cubemap [C, dim, 6*dim] with faces
    [-z, -x, +z, +x, +y, -y] -> equirectangular [C, rect_height, rect_width]."""
    _contig(cubemap=cubemap)
    _on_gpu("cubemap", cubemap)
    if cubemap.dtype not in (torch.float32, torch.float64):
        raise RuntimeError("unsupported dtype %s" % cubemap.dtype)
    if cubemap.dim() != 3 or cubemap.shape[2] != 6 * cubemap.shape[1]:
        raise RuntimeError("cubemap must be [C, dim, 6*dim], got %s" % (tuple(cubemap.shape),))
    C, dim = cubemap.shape[0], cubemap.shape[1]
    RH, RW = int(rect_height), int(rect_width)
    rect = torch.empty((C, RH, RW), dtype=cubemap.dtype, device=cubemap.device)
    with _device(cubemap):
        rc = _lib.load().mcx_cube2rect(_ptr(cubemap), _ptr(rect), C, dim, RH, RW,
                                       int(interpolation), _DTYPES[cubemap.dtype],
                                       _stream(cubemap))
    _lib.check(rc, "cube2rect")
    return rect


# ------------------------------------------------------------ icosphere map operators
def gnomonic_samples(centres, kh, kw, res_lat, res_lon):
    """gnomonic_kernel of package/layers/util/icosphere_functions.py:135-183 on the device:
    centres [V, 2] (longitude, latitude), float32 -> [1, V, kh*kw, 2]."""
    _contig(centres=centres)
    _on_gpu("spherical_coords", centres)
    if centres.dtype != torch.float32 or centres.dim() != 2 or centres.shape[1] != 2:
        raise RuntimeError("spherical_coords must be a float32 tensor [V, 2]")
    V = centres.shape[0]
    out = torch.empty((1, V, int(kh) * int(kw), 2), dtype=torch.float32, device=centres.device)
    with _device(centres):
        rc = _lib.load().mcx_gnomonic_samples(_ptr(centres), _ptr(out), V, int(kh), int(kw),
                                              float(res_lat), float(res_lon), _stream(centres))
    _lib.check(rc, "gnomonic_kernel")
    return out


def planar_conv_operator_from_samples(samples, vertices, faces, keepdim=True, nearest=False):
    """Sphere.get_planar_conv_operator_from_samples of the reference's `_sphere` module
    (package/ext_modules/src/util/cpp/sphere.cpp:1117-1270) over a caller-supplied mesh.

    samples [OH, OW, K, 2] or [OH, OW, 2] (longitude, latitude), float32, on the GPU;
    vertices [V, 3] float32 and faces [F, 3] int64 of a closed triangle mesh around the
    origin.  Returns [face_idx [OH, OW, K] int64, vertex_idx [OH, OW, K, 3] int64,
    weights [OH, OW, K, 3] float32]; a [OH, OW, 2] input without `keepdim` drops the K axis,
    as in the reference."""
    _contig(samples=samples, vertices=vertices, faces=faces)
    _on_gpu("samples", samples, vertices=vertices, faces=faces)
    if samples.dtype != torch.float32 or vertices.dtype != torch.float32:
        raise RuntimeError("samples and vertices must be float32")
    if faces.dtype != torch.int64:
        raise RuntimeError("faces must be int64")
    if samples.dim() not in (3, 4) or samples.shape[-1] != 2:
        raise RuntimeError("samples must be [OH, OW, K, 2] or [OH, OW, 2]")
    if vertices.dim() != 2 or vertices.shape[1] != 3 or faces.dim() != 2 or faces.shape[1] != 3:
        raise RuntimeError("vertices must be [V, 3] and faces [F, 3]")
    lead = tuple(samples.shape[:-1])
    if samples.dim() == 3 and keepdim:
        lead = lead + (1,)
    N, V, F = samples.numel() // 2, vertices.shape[0], faces.shape[0]
    dev = samples.device
    face_idx = torch.empty(lead, dtype=torch.int64, device=dev)
    vertex_idx = torch.empty(lead + (3,), dtype=torch.int64, device=dev)
    weights = torch.empty(lead + (3,), dtype=torch.float32, device=dev)
    lib = _lib.load()
    ws_bytes = lib.mcx_planar_conv_operator_workspace(F)
    ws = _workspace(ws_bytes, dev)
    with torch.cuda.device(dev):
        rc = lib.mcx_planar_conv_operator(_ptr(samples), _ptr(vertices), _ptr(faces),
                                          _ptr(face_idx), _ptr(vertex_idx), _ptr(weights),
                                          _ptr(ws), ws_bytes, N, V, F, 1 if nearest else 0,
                                          _stream(samples))
    _lib.check(rc, "planar_conv_operator_from_samples")
    return [face_idx, vertex_idx, weights]


# ---- attention with a bias by relative-position buckets, and what goes with it -------------
# (no counterpart in the reference)

def _attention_dtype(data, **same):
    """Data type code of the attention operators: float32 or bfloat16, one for all operands."""
    if data.dtype != torch.float32 and data.dtype != torch.bfloat16:
        raise RuntimeError("unsupported dtype %s (float32 or bfloat16)" % data.dtype)
    for name, t in same.items():
        if t is not None and t.dtype != data.dtype:
            raise RuntimeError("%s is %s, expected %s" % (name, t.dtype, data.dtype))
    return _DTYPES[data.dtype]


def _heads(name, t, B=None, L=None, H=None, D=None):
    """Shape of a [B, L, H, D] tensor, after a check of the sizes that are given."""
    shape = t.shape
    if len(shape) != 4:
        raise RuntimeError("%s must have 4 dimensions [B, L, H, D], got %s" % (name, tuple(shape)))
    for axis, want in enumerate((B, L, H, D)):
        if want is not None and shape[axis] != want:
            raise RuntimeError("%s has size %d in dimension %d, expected %d" %
                               (name, shape[axis], axis, want))
    return shape


def _dense_last(t):
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


def _norm_args(query, key, query_weight, key_weight, cos, sin, positions, eps):
    B, L, Hq, D = _heads("query", query)
    _, _, Hk, _ = _heads("key", key, B, L, None, D)
    dt = _attention_dtype(query, key=key, query_weight=query_weight, key_weight=key_weight)
    _on_gpu("query", query, key=key, query_weight=query_weight, key_weight=key_weight, cos=cos,
            sin=sin, positions=positions)
    if Hq < 1 or Hk < 1 or not 1 <= D <= 256:
        raise RuntimeError("heads of 1 to 256 values are supported (got %d heads, %d key heads, "
                           "%d values)" % (Hq, Hk, D))
    for name, w in (("query_weight", query_weight), ("key_weight", key_weight)):
        if tuple(w.shape) != (D,):
            raise RuntimeError("%s must have shape (%d,), got %s" % (name, D, tuple(w.shape)))
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise RuntimeError("cos and sin must be float32")
    if cos.dim() != 2 or cos.shape != sin.shape or 2 * cos.shape[1] > D:
        raise RuntimeError("cos and sin must have the same shape [places, F] with 2 F <= %d, got "
                           "%s and %s" % (D, tuple(cos.shape), tuple(sin.shape)))
    if positions is not None:
        if positions.dtype != torch.int64 or tuple(positions.shape) != (B, L):
            raise RuntimeError("positions must be int64 of shape (%d, %d), got %s %s" %
                               (B, L, positions.dtype, tuple(positions.shape)))
        positions = positions.contiguous()
    elif cos.shape[0] < L:
        raise RuntimeError("cos and sin have %d places for %d positions" % (cos.shape[0], L))
    if not eps >= 0:
        raise RuntimeError("eps must not be negative")
    _contig(query_weight=query_weight, key_weight=key_weight)
    return (dt, B, L, Hq, Hk, D, _dense_last(query), _dense_last(key), cos.contiguous(),
            sin.contiguous(), positions)


_three = _lib._i64 * 3


def _strides(t):
    return _three(*t.stride()[:3])


def qk_norm_rotate_forward(query, key, query_weight, key_weight, cos, sin, positions=None,
                           eps=1e-6, adjacent=False):
    """Queries [B, L, Hq, D] and keys [B, L, Hk, D] (views of a packed projection go as they are),
    every head of every token divided by its root mean square and multiplied by query_weight /
    key_weight [D]; then the first 2 F values of each turned by the angles of the token's place:
    cos, sin float32 [places, F], the place being `positions` [B, L] (int64) or the index along
    L.  A pair is (f, f + F), or (2 f, 2 f + 1) if `adjacent`.  -> [query, key], contiguous.
    A position outside the places gives NaN."""
    dt, B, L, Hq, Hk, D, query, key, cos, sin, positions = _norm_args(
        query, key, query_weight, key_weight, cos, sin, positions, eps)
    q_out, k_out = query.new_empty((B, L, Hq, D)), query.new_empty((B, L, Hk, D))
    with _device(query):
        rc = _lib.load().mcx_qk_norm_rotate_forward(
            _ptr(query), _ptr(key), _ptr(query_weight), _ptr(key_weight), _ptr(cos), _ptr(sin),
            _ptr(positions), _ptr(q_out), _ptr(k_out), _strides(query), _strides(key), B, L, Hq,
            Hk, D, cos.shape[1], cos.shape[0], float(eps), int(bool(adjacent)), dt, _stream(query))
    _lib.check(rc, "qk_norm_rotate_forward")
    return [q_out, k_out]


def qk_norm_rotate_backward(grad_query, grad_key, query, key, query_weight, key_weight, cos, sin,
                            positions=None, eps=1e-6, adjacent=False,
                            needs=(True, True, True, True)):
    """-> [grad_query, grad_key, grad_query_weight, grad_key_weight] of qk_norm_rotate_forward
    from the gradients of its outputs; a gradient that `needs` leaves out is None."""
    dt, B, L, Hq, Hk, D, query, key, cos, sin, positions = _norm_args(
        query, key, query_weight, key_weight, cos, sin, positions, eps)
    _heads("grad_query", grad_query, B, L, Hq, D)
    _heads("grad_key", grad_key, B, L, Hk, D)
    _attention_dtype(query, grad_query=grad_query, grad_key=grad_key)
    _on_gpu("query", query, grad_query=grad_query, grad_key=grad_key)
    grad_query, grad_key = grad_query.contiguous(), grad_key.contiguous()
    gq, gk, gwq, gwk = (torch.empty_like(t) if wanted else None for t, wanted in
                        zip((grad_query, grad_key, query_weight, key_weight), needs))
    lib = _lib.load()
    nbytes = lib.mcx_qk_norm_rotate_backward_workspace(B, L, Hq, Hk, D, dt)
    ws = _workspace(nbytes, query.device)
    with _device(query):
        rc = lib.mcx_qk_norm_rotate_backward(
            _ptr(grad_query), _ptr(grad_key), _ptr(query), _ptr(key), _ptr(query_weight),
            _ptr(key_weight), _ptr(cos), _ptr(sin), _ptr(positions), _ptr(gq), _ptr(gk), _ptr(gwq),
            _ptr(gwk), _ptr(ws), nbytes, _strides(query), _strides(key), B, L, Hq, Hk, D,
            cos.shape[1], cos.shape[0], float(eps), int(bool(adjacent)), dt, _stream(query))
    _lib.check(rc, "qk_norm_rotate_backward")
    return [gq, gk, gwq, gwk]


def _attention_args(query, key, value, bias_table, buckets, bucket_zero, scale, causal,
                    query_start, key_lengths):
    """(dtype code, descriptor, the tensors as the library takes them) of an attention call."""
    B, Lq, Hq, D = _heads("query", query)
    _, Lk, Hk, _ = _heads("key", key, B, None, None, D)
    _heads("value", value, B, Lk, Hk, D)
    dt = _attention_dtype(query, key=key, value=value, bias_table=bias_table)
    _on_gpu("query", query, key=key, value=value, bias_table=bias_table, buckets=buckets,
            query_start=query_start, key_lengths=key_lengths)
    if Hk < 1 or Hq % Hk or Hq < 1:
        raise RuntimeError("%d query heads cannot share %d key heads" % (Hq, Hk))
    if not 1 <= D <= 128:
        raise RuntimeError("heads of 1 to 128 values are supported, got %d" % D)
    if (bias_table is None) != (buckets is None):
        raise RuntimeError("bias_table and buckets go together")
    if bias_table is not None:
        if bias_table.dim() != 2 or bias_table.shape[0] != Hq or \
                not 1 <= bias_table.shape[1] <= 512:
            raise RuntimeError("bias_table must be [%d, 1 to 512 buckets], got %s" %
                               (Hq, tuple(bias_table.shape)))
        if buckets.dtype != torch.int32 or buckets.dim() != 1:
            raise RuntimeError("buckets must be a vector of int32, got %s %s" %
                               (buckets.dtype, tuple(buckets.shape)))
        if not 0 <= bucket_zero < buckets.shape[0]:
            raise RuntimeError("bucket_zero %d is no entry of %d buckets" %
                               (bucket_zero, buckets.shape[0]))
        bias_table, buckets = bias_table.contiguous(), buckets.contiguous()
    for name, t in (("query_start", query_start), ("key_lengths", key_lengths)):
        if t is not None and (t.dtype != torch.int32 or tuple(t.shape) != (B,)):
            raise RuntimeError("%s must be int32 of shape (%d,), got %s %s" %
                               (name, B, t.dtype, tuple(t.shape)))
    scale = D ** -0.5 if scale is None else float(scale)
    if not 1e-6 <= scale <= 1e6:
        raise RuntimeError("scale must lie between 1e-6 and 1e6, got %g" % scale)
    query, key, value = _dense_last(query), _dense_last(key), _dense_last(value)
    if query_start is not None:
        query_start = query_start.contiguous()
    if key_lengths is not None:
        key_lengths = key_lengths.contiguous()
    n, size = (0, 0) if bias_table is None else (buckets.shape[0], bias_table.shape[1])
    desc = _lib.AttentionDesc(B, Lq, Lk, Hq, Hk, D, _strides(query), _strides(key),
                              _strides(value), n, int(bucket_zero) if n else 0, size, scale,
                              int(bool(causal)), 0)
    return dt, desc, (query, key, value, bias_table, buckets, query_start, key_lengths)


def relative_attention_forward(query, key, value, bias_table=None, buckets=None, bucket_zero=0,
                               scale=None, causal=False, query_start=None, key_lengths=None,
                               for_backward=False):
    """Attention of queries [B, Lq, Hq, D] over keys and values [B, Lk, Hk, D] (Hk divides Hq;
    any strides with a dense last axis) with a learned bias by relative position:

        out = softmax_j(scale q_i . k_j + bias_table[h, buckets[clamp(j - pos_i + bucket_zero)]]) v_j

    query i standing at position pos_i = query_start[b] + i (0 + i by default) and key j at j.
    bias_table [Hq, buckets of a head]; buckets int32, one entry a difference, the ends standing
    for all beyond.  `causal` keeps the keys up to the query's own position; key_lengths int32 [B]
    says how many keys are in use: what lies behind them is not read.  scale: D ** -0.5 by default.
    A row that nothing is left of is zeros.  A bucket that the table does not have has no bias; a
    bias of -inf takes its pairs out.
    -> [out [B, Lq, Hq, D], saved]: `saved`, for relative_attention_backward, is None unless
    `for_backward`: a list of the rows' statistics (float32) and, for bfloat16, of what rounding took
    from the output.  Keys and values within key_lengths have to be finite."""
    dt, desc, tensors = _attention_args(query, key, value, bias_table, buckets, bucket_zero, scale,
                                        causal, query_start, key_lengths)
    query = tensors[0]
    B, Lq, Hq, D = query.shape
    out = query.new_empty((B, Lq, Hq, D))
    stats = rest = None
    if for_backward:
        stats = torch.empty((B, Hq, Lq, 2), dtype=torch.float32, device=query.device)
        rest = torch.empty_like(out) if dt == MCX_BF16 else None
    lib = _lib.load()
    nbytes = lib.mcx_attention_forward_workspace(desc, dt)
    ws = _workspace(nbytes, query.device) if nbytes else None
    with _device(query):
        rc = lib.mcx_attention_forward(*[_ptr(t) for t in tensors], _ptr(out), _ptr(stats),
                                       _ptr(rest), _ptr(ws), nbytes, desc, dt, _stream(query))
    _lib.check(rc, "relative_attention_forward")
    return [out, [stats, rest] if for_backward else None]


def relative_attention_backward(grad_output, query, key, value, output, saved, bias_table=None,
                                buckets=None, bucket_zero=0, scale=None, causal=False,
                                query_start=None, key_lengths=None,
                                needs=(True, True, True, True)):
    """-> [grad_query, grad_key, grad_value, grad_bias_table] of relative_attention_forward, called
    with the same arguments and `for_backward`; a gradient that `needs` leaves out is None.  The
    same bits from call to call."""
    dt, desc, tensors = _attention_args(query, key, value, bias_table, buckets, bucket_zero, scale,
                                        causal, query_start, key_lengths)
    query, key, value, table = tensors[:4]
    _heads("grad_output", grad_output, *query.shape)
    _heads("output", output, *query.shape)
    _attention_dtype(query, grad_output=grad_output, output=output)
    B, Lq, Hq, D = query.shape
    stats, rest = saved if saved is not None else (None, None)
    if stats is None or stats.dtype != torch.float32 or tuple(stats.shape) != (B, Hq, Lq, 2) or \
            (rest is not None and (rest.dtype != query.dtype or rest.shape != query.shape)):
        raise RuntimeError("saved must be what relative_attention_forward returned with for_backward")
    _on_gpu("query", query, grad_output=grad_output, output=output, stats=stats, rest=rest)
    _contig(stats=stats, rest=rest)
    grad_output, output = grad_output.contiguous(), output.contiguous()

    def like(t, wanted):
        return torch.empty(t.shape, dtype=t.dtype, device=t.device) if wanted else None

    gq, gk, gv = like(query, needs[0]), like(key, needs[1]), like(value, needs[2])
    gt = like(table, needs[3]) if table is not None else None
    if B == 0 or Lq == 0:
        for t in (gk, gv, gt):
            if t is not None:
                t.zero_()
        return [gq, gk, gv, gt]
    lib = _lib.load()
    nbytes = lib.mcx_attention_backward_workspace(desc, dt)
    ws = _workspace(nbytes, query.device)
    with _device(query):
        rc = lib.mcx_attention_backward(_ptr(grad_output), *[_ptr(t) for t in tensors[:3]],
                                        _ptr(output), _ptr(rest), _ptr(stats),
                                        *[_ptr(t) for t in tensors[3:]],
                                        _ptr(gq), _ptr(gk), _ptr(gv), _ptr(gt), _ptr(ws), nbytes,
                                        desc, dt, _stream(query))
    _lib.check(rc, "relative_attention_backward")
    return [gq, gk, gv, gt]


_CLIP_DTYPES = {torch.float32: MCX_F32, torch.bfloat16: MCX_BF16}


def _written_apart(read, write, tensors):
    """Refuses a tensor that would be written while another one's work reads or writes it."""
    # (tensors without values may share an address)
    pairs = [(r, w) for r, w, t in zip(read, write, tensors) if t.numel()]
    if len({w for _, w in pairs}) != len(pairs):
        raise RuntimeError("a tensor that is written stands in the list twice")
    if not {w for r, w in pairs if r != w}.isdisjoint(r for r, _ in pairs):
        raise RuntimeError("a tensor of out is another one's input")


def clip_grad_norm(tensors, max_norm, eps=1e-6, out=None):
    """The norm of all values of a list of tensors (float32 and bfloat16, contiguous, on one GPU),
    as a float32 scalar; the tensors, or where `out` gives as many of the same sizes and types
    those, hold min(1, max_norm / (norm + eps)) times the values then.  A norm that is no number
    makes them all none.  What is written must not share memory with any other tensor: one that
    stands in the list twice is refused, parts that overlap are not looked for."""
    max_norm, eps = float(max_norm), float(eps)
    if not max_norm >= 0 or not eps >= 0:
        raise RuntimeError("max_norm and eps must not be negative")
    tensors = list(tensors)
    if not tensors:
        raise RuntimeError("clip_grad_norm needs at least one tensor")
    # (hundreds of tensors: every look at them is one pass in C)
    every, n = tensors if out is None else tensors + list(out), len(tensors)
    if len(every) != (n if out is None else 2 * n):
        raise RuntimeError("out must have as many tensors")
    at = list(map(torch.Tensor.data_ptr, every))
    if len(set(at)) != len(at):
        _written_apart(at[:n], at[-n:], tensors)
    where = set(map(torch.Tensor.get_device, every))
    if len(where) != 1 or not tensors[0].is_cuda:
        raise RuntimeError("all tensors must be on one GPU")
    if not all(map(torch.Tensor.is_contiguous, every)):
        raise RuntimeError("tensors must be contiguous")
    sizes = list(map(torch.Tensor.numel, every))
    codes = [_CLIP_DTYPES.get(t.dtype, -1) for t in every]
    if -1 in codes:
        raise RuntimeError("unsupported dtype %s (float32 or bfloat16)" % every[codes.index(-1)].dtype)
    if out is not None and (sizes[:n] != sizes[n:] or codes[:n] != codes[n:]):
        raise RuntimeError("out must have the tensors' sizes and dtypes")
    # (host arrays of the library's types; `inputs` and the others live until it has returned)
    inputs, outputs = array.array("Q", at[:n]), array.array("Q", at[-n:])
    lengths, types = array.array("q", sizes[:n]), array.array("i", codes[:n])
    hosts = [a.buffer_info()[0] for a in (inputs, outputs, lengths, types)]
    device = tensors[0].device
    lib = _lib.load()
    norm = torch.empty((), dtype=torch.float32, device=device)
    nbytes = lib.mcx_clip_grad_norm_workspace(hosts[2], n)
    ws = _workspace(nbytes, device)
    with _device(norm):
        rc = lib.mcx_clip_grad_norm(*hosts, n, max_norm, eps, _ptr(norm), _ptr(ws), nbytes,
                                    _stream(norm))
    _lib.check(rc, "clip_grad_norm")
    _changed(every[-n:])
    return norm


# ---- a gated linear recurrence along a sequence ---------------------------------------------

_two = _lib._i64 * 2
_RECURRENCE_STRIDE = 1 << 22


def _recurrence_args(value, forget, gate, lengths, reverse, states=(), **others):
    """(dtype code, descriptor, the tensors as the library takes them) of a recurrence call; `states`:
    the names of those of the others that are states."""
    shape = value.shape
    if len(shape) != 3 or shape[2] < 1:
        raise RuntimeError("value must have 3 dimensions [B, L, C], got %s" % (tuple(shape),))
    for name, t in (("forget", forget), ("gate", gate)):
        if t is not None and t.shape != shape:
            raise RuntimeError("%s must have value's shape %s, got %s" %
                               (name, tuple(shape), tuple(t.shape)))
    dt = _attention_dtype(value, forget=forget, gate=gate)
    _on_gpu("value", value, forget=forget, gate=gate, lengths=lengths, **others)
    B, L, C = shape
    for name in states:
        t = others[name]
        if t is not None and (t.dtype != torch.float32 or t.shape != (B, C)):
            raise RuntimeError("%s must be float32 of shape (%d, %d), got %s %s" %
                               (name, B, C, t.dtype, tuple(t.shape)))
    if lengths is not None:
        if lengths.dtype != torch.int32 or tuple(lengths.shape) != (B,):
            raise RuntimeError("lengths must be int32 of shape (%d,), got %s %s" %
                               (B, lengths.dtype, tuple(lengths.shape)))
        lengths = lengths.contiguous()
    # (steps further apart than the kernels' addresses reach are copied)
    tensors, strides = [], []
    for t in (value, forget, gate):
        stride = (0, 0, 1) if t is None else t.stride()
        if (stride[2] != 1 and C != 1) or stride[1] > _RECURRENCE_STRIDE:
            t = t.contiguous()
            stride = t.stride()
        tensors.append(t)
        strides.append(stride[:2])
    desc = _lib.RecurrenceDesc(B, L, C, *strides, int(bool(reverse)), 0)
    return (dt, desc, *tensors, lengths)


def gated_recurrence_forward(value, forget, gate=None, initial=None, lengths=None, reverse=False,
                             final=None, for_backward=False):
    """A linear recurrence of every channel along the sequence, value, forget and gate [B, L, C] (any
    strides with a dense last axis; parts of one projection go as they are):

        a_t = sigmoid(forget_t),   h_t = a_t h_{t-1} + (1 - a_t) value_t
        out_t = h_t gate_t sigmoid(gate_t)                          (h_t without a gate)

    from the state `initial` float32 [B, C] (zeros by default).  lengths int32 [B] says how many steps
    are in use: what lies behind them is not read, and out is zero there; `reverse` takes them from the
    last one in use to the first.
    -> [out [B, L, C], final, saved]: the state after the last step float32 [B, C], in the tensor `final`
    where one is given (it may be `initial`, for a state that is kept from call to call); `saved`, for
    gated_recurrence_backward, is None unless `for_backward`: states at some of the steps, float32."""
    dt, desc, value, forget, gate, lengths = _recurrence_args(
        value, forget, gate, lengths, reverse, ("initial", "final"), initial=initial, final=final)
    B, L, C = value.shape
    _contig(final=final)
    if initial is not None:
        initial = initial.contiguous()
    out = value.new_empty((B, L, C))
    given = final is not None
    if not given:
        final = torch.empty((B, C), dtype=torch.float32, device=value.device)
    lib = _lib.load()
    states = None
    if for_backward:
        states = torch.empty((B, lib.mcx_gated_recurrence_spans(L), C), dtype=torch.float32,
                             device=value.device)
    if B and not L:  # no step: the state stays as it is
        if initial is None:
            final.zero_()
        elif final.data_ptr() != initial.data_ptr():
            final.copy_(initial)
    nbytes = lib.mcx_gated_recurrence_workspace(desc, dt)
    ws = _workspace(nbytes, value.device) if nbytes else None
    with _device(value):
        rc = lib.mcx_gated_recurrence_forward(_ptr(value), _ptr(forget), _ptr(gate), _ptr(initial),
                                              _ptr(lengths), _ptr(out), _ptr(final), _ptr(states),
                                              _ptr(ws), nbytes, desc, dt, _stream(value))
    _lib.check(rc, "gated_recurrence_forward")
    if given:
        _changed(final)
    return [out, final, states]


def gated_recurrence_backward(grad_output, value, forget, gate, saved, grad_final=None, lengths=None,
                              reverse=False, needs=(True, True, True, True)):
    """-> [grad_value, grad_forget, grad_gate, grad_initial] of gated_recurrence_forward, called with the
    same arguments and `for_backward`, from the gradients of out and (float32, zeros by default) of
    final; a gradient that `needs` leaves out, or that of a gate that there is not, is None.  The same
    bits from call to call."""
    dt, desc, value, forget, gate, lengths = _recurrence_args(
        value, forget, gate, lengths, reverse, ("grad_final",), grad_final=grad_final,
        grad_output=grad_output, saved=saved)
    B, L, C = value.shape
    lib = _lib.load()
    if grad_output.shape != value.shape:
        raise RuntimeError("grad_output must have shape %s, got %s" %
                           (tuple(value.shape), tuple(grad_output.shape)))
    _attention_dtype(value, grad_output=grad_output)
    if saved is None or saved.dtype != torch.float32 or \
            tuple(saved.shape) != (B, lib.mcx_gated_recurrence_spans(L), C):
        raise RuntimeError("saved must be what gated_recurrence_forward returned with for_backward")
    _contig(saved=saved)
    grad_output = grad_output.contiguous()
    if grad_final is not None:
        grad_final = grad_final.contiguous()
    gv, gf, gg = (value.new_empty((B, L, C)) if wanted and t is not None else None
                  for t, wanted in zip((value, forget, gate), needs))
    gi = torch.empty((B, C), dtype=torch.float32, device=value.device) if needs[3] else None
    if B and not L and gi is not None:
        gi.zero_() if grad_final is None else gi.copy_(grad_final)
    if not any(needs):
        return [None, None, None, None]
    nbytes = lib.mcx_gated_recurrence_workspace(desc, dt)
    ws = _workspace(nbytes, value.device) if nbytes else None
    with _device(value):
        rc = lib.mcx_gated_recurrence_backward(
            _ptr(grad_output), _ptr(grad_final), _ptr(value), _ptr(forget), _ptr(gate), _ptr(saved),
            _ptr(lengths), _ptr(gv), _ptr(gf), _ptr(gg), _ptr(gi), _ptr(ws), nbytes, desc, dt,
            _stream(value))
    _lib.check(rc, "gated_recurrence_backward")
    return [gv, gf, gg, gi]


# ---- group norm with an activation, channels last -----------------------------------------

ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2}


def _group_args(x, groups, weight, bias, activation):
    shape = x.shape
    if len(shape) != 3:
        raise RuntimeError("x must have 3 dimensions [B, N, C], got %s" % (tuple(shape),))
    dt = _attention_dtype(x, weight=weight, bias=bias)
    _on_gpu("x", x, weight=weight, bias=bias)
    groups = int(groups)
    if groups < 1 or shape[2] < 1 or shape[2] % groups:
        raise RuntimeError("%d channels cannot be cut into %d groups" % (shape[2], groups))
    if activation not in ACTIVATIONS:
        raise RuntimeError("activation must be one of %s, got %r" %
                           (", ".join(map(repr, ACTIVATIONS)), activation))
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and tuple(t.shape) != (shape[2],):
            raise RuntimeError("%s must have shape (%d,), got %s" % (name, shape[2], tuple(t.shape)))
    _contig(weight=weight, bias=bias)
    if x.stride(2) != 1 and shape[2] != 1:
        x = x.contiguous()
    return dt, groups, ACTIVATIONS[activation], x


def group_norm_forward(x, groups, weight=None, bias=None, eps=1e-5, activation=None,
                       for_backward=False):
    """x [B, N, C] (any strides with a dense last axis), every group of C / groups neighbouring channels of
    a sample normed over the N tokens: y = act((x - mean) / sqrt(var + eps) * weight + bias), weight and
    bias [C]; activation None, "silu" (u / (1 + e^-u)) or "gelu" (u (1 + erf(u / sqrt 2)) / 2).
    -> [y, saved], y contiguous; `saved`, for group_norm_backward, is None unless `for_backward`:
    mean and 1 / sqrt(var + eps) of every group, float32 [B, groups, 2]."""
    dt, groups, act, x = _group_args(x, groups, weight, bias, activation)
    eps = float(eps)
    if not eps >= 0:
        raise RuntimeError("eps must not be negative")
    B, N, C = x.shape
    y = x.new_empty((B, N, C))
    stats = torch.empty((B, groups, 2), dtype=torch.float32, device=x.device) if for_backward else None
    lib = _lib.load()
    nbytes = lib.mcx_group_norm_workspace(B, N, C, groups, 0, dt)
    ws = _workspace(nbytes, x.device)
    with _device(x):
        rc = lib.mcx_group_norm_forward(_ptr(x), _ptr(weight), _ptr(bias), _ptr(y), _ptr(stats),
                                        _ptr(ws), nbytes, _two(*x.stride()[:2]), B, N, C,
                                        groups, eps, act, dt, _stream(x))
    _lib.check(rc, "group_norm_forward")
    return [y, stats]


def group_norm_backward(grad_output, x, saved, groups, weight=None, bias=None, activation=None,
                        needs=(True, True, True)):
    """-> [grad_x, grad_weight, grad_bias] of group_norm_forward from the gradient of y and what it
    saved; a gradient that `needs` leaves out, or whose parameter there is not, is None.  The same
    bits from call to call."""
    dt, groups, act, x = _group_args(x, groups, weight, bias, activation)
    B, N, C = x.shape
    if tuple(grad_output.shape) != (B, N, C):
        raise RuntimeError("grad_output must have shape (%d, %d, %d), got %s" %
                           (B, N, C, tuple(grad_output.shape)))
    _attention_dtype(x, grad_output=grad_output)
    if saved is None or saved.dtype != torch.float32 or tuple(saved.shape) != (B, groups, 2):
        raise RuntimeError("saved must be what group_norm_forward returned with for_backward")
    _on_gpu("x", x, grad_output=grad_output, saved=saved)
    _contig(saved=saved)
    grad_output = grad_output.contiguous()
    gx = x.new_empty((B, N, C)) if needs[0] else None
    gw = torch.empty_like(weight) if weight is not None and needs[1] else None
    gb = torch.empty_like(bias) if bias is not None and needs[2] else None
    if B == 0 or N == 0:
        for t in (gw, gb):
            if t is not None:
                t.zero_()
        return [gx, gw, gb]
    lib = _lib.load()
    nbytes = lib.mcx_group_norm_workspace(B, N, C, groups, 1, dt)
    ws = _workspace(nbytes, x.device)
    with _device(x):
        rc = lib.mcx_group_norm_backward(_ptr(grad_output), _ptr(x), _ptr(saved), _ptr(weight),
                                         _ptr(bias), _ptr(gx), _ptr(gw), _ptr(gb), _ptr(ws), nbytes,
                                         _two(*x.stride()[:2]), B, N, C, groups, act, dt,
                                         _stream(x))
    _lib.check(rc, "group_norm_backward")
    return [gx, gw, gb]


# ---- clipping's norm alone, and the AdamW step ------------------------------------------------

def _together(tensors):
    """Addresses and sizes (lists) of tensors that have to be contiguous and on one GPU."""
    # (hundreds of tensors: every look at them is one pass in C)
    if len(set(map(torch.Tensor.get_device, tensors))) != 1 or not tensors[0].is_cuda:
        raise RuntimeError("all tensors must be on one GPU")
    if not all(map(torch.Tensor.is_contiguous, tensors)):
        raise RuntimeError("tensors must be contiguous")
    return list(map(torch.Tensor.data_ptr, tensors)), list(map(torch.Tensor.numel, tensors))


def _type_codes(dtypes):
    codes = list(map(_CLIP_DTYPES.get, dtypes))
    if None in codes:
        raise RuntimeError("unsupported dtype %s (float32 or bfloat16)" % dtypes[codes.index(None)])
    return array.array("i", codes)


def grad_norm(tensors):
    """The norm of all values of a list of tensors (float32 and bfloat16, contiguous, on one GPU), as
    a float32 scalar; what clip_grad_norm multiplies by, without the products: adamw_step takes it."""
    tensors = list(tensors)
    if not tensors:
        raise RuntimeError("grad_norm needs at least one tensor")
    at, sizes = _together(tensors)
    types = _type_codes([t.dtype for t in tensors])
    # (host arrays of the library's types, which live until it has returned)
    at, sizes = array.array("Q", at), array.array("q", sizes)
    hosts = [a.buffer_info()[0] for a in (at, sizes, types)]
    device = tensors[0].device
    lib = _lib.load()
    norm = torch.empty((), dtype=torch.float32, device=device)
    nbytes = lib.mcx_clip_grad_norm_workspace(hosts[1], len(tensors))
    ws = _workspace(nbytes, device)
    with _device(norm):
        rc = lib.mcx_clip_grad_norm(hosts[0], None, hosts[1], hosts[2], len(tensors), 0.0, 0.0,
                                    _ptr(norm), _ptr(ws), nbytes, _stream(norm))
    _lib.check(rc, "grad_norm")
    return norm


ADAMW_BLOCK = 256  # values that share a scale where moments are held in 8 bits


def _one_value(name, t, dtype, like):
    if t.dtype != dtype or t.numel() != 1 or t.get_device() != like.get_device():
        raise RuntimeError("%s must be one %s value on the parameters' GPU" % (name, dtype))
    return t.data_ptr()


def adamw_step(params, grads, first_moments, second_moments, step, lr, betas=(0.9, 0.999), eps=1e-8,
               weight_decay=0.0, first_scales=None, second_scales=None, seed=0, grad_norm=None,
               max_norm=None):
    """One AdamW step over lists of tensors on one GPU, in place:

        g' = g min(1, max_norm / (grad_norm + 1e-6))        (g without grad_norm and max_norm)
        m = b1 m + (1 - b1) g',   v = b2 v + (1 - b2) g'^2
        p = p (1 - lr weight_decay) - lr / (1 - b1^step) m / (sqrt(v) / sqrt(1 - b2^step) + eps)

    Parameters and gradients are float32 or bfloat16, each of its own type, contiguous.  The moments are
    float32; or, with scales, uint8, which 256 values of a tensor share a float32 scale of
    (first_scales, second_scales: (size + 255) // 256 values a tensor; zeros at the start): 3 bits
    and an exponent each, rounded up with the probability of what is cut off, by words that `seed`, the
    step and the value's place in the list give.
    step: the number of this step from 1 on, or an int64 value on the GPU; lr: a number, or a float32
    value on the GPU; both are read there when the kernels run, so that a captured step can be replayed.
    What is changed must not share memory with any other tensor: one that stands in the lists twice
    is refused, parts that overlap are not looked for."""
    _adamw_call(params, grads, first_moments, second_moments, step, lr, betas, eps, weight_decay,
                first_scales, second_scales, seed, grad_norm, max_norm)()


def _adamw_call(params, grads, first_moments, second_moments, step, lr, betas, eps, weight_decay,
                first_scales=None, second_scales=None, seed=0, grad_norm=None, max_norm=None):
    """adamw_step's checks -> what launches the step, so that a caller can have several steps checked before
    the first of them changes anything."""
    if (first_scales is None) != (second_scales is None):
        raise RuntimeError("first_scales and second_scales go together")
    if (grad_norm is None) != (max_norm is None):
        raise RuntimeError("grad_norm and max_norm go together")
    beta1, beta2 = betas
    max_norm = 0.0 if max_norm is None else float(max_norm)
    if not (0 <= beta1 < 1 and 0 <= beta2 < 1 and eps >= 0 and weight_decay >= 0 and max_norm >= 0):
        raise RuntimeError("betas must lie in [0, 1), eps, weight_decay and max_norm must not be "
                           "negative")
    on_gpu = isinstance(step, torch.Tensor), isinstance(lr, torch.Tensor)
    if not on_gpu[0] and int(step) < 1:
        raise RuntimeError("step counts from 1, got %d" % step)
    if not on_gpu[1] and not abs(float(lr)) < float("inf"):
        raise RuntimeError("lr must be finite")
    lists = [list(params), list(grads), list(first_moments), list(second_moments)]
    wide = first_scales is None
    if not wide:
        lists += [list(first_scales), list(second_scales)]
    n = len(lists[0])
    if set(map(len, lists)) != {n}:
        raise RuntimeError("every list must have as many tensors: %s" % list(map(len, lists)))
    if not n:
        return lambda: None
    every = sum(lists, [])
    at, sizes = _together(every)
    dtypes = [t.dtype for t in every]
    types = _type_codes(dtypes[:2 * n])
    if set(dtypes[2 * n:4 * n]) != {torch.float32 if wide else torch.uint8}:
        raise RuntimeError("moments must be float32, or uint8 with scales")
    if set(dtypes[4 * n:]) - {torch.float32}:
        raise RuntimeError("scales must be float32")
    if sizes[:n] * 3 != sizes[n:4 * n]:
        raise RuntimeError("gradients and moments must have the parameters' sizes")
    if not wide and [-(-k // ADAMW_BLOCK) for k in sizes[:n]] * 2 != sizes[4 * n:]:
        raise RuntimeError("there must be one scale for %d values of a tensor" % ADAMW_BLOCK)
    written = at[:n] + at[2 * n:]
    places = set(written)
    if len(places) != len(written) or not places.isdisjoint(at[n:2 * n]):
        # (tensors without values may share an address)
        full = [a for a, k in zip(written, sizes[:n] + sizes[2 * n:]) if k]
        if len(set(full)) != len(full) or \
                not set(full).isdisjoint(a for a, k in zip(at[n:2 * n], sizes) if k):
            raise RuntimeError("a tensor that is changed stands in the lists twice")
    first = every[0]
    options = _lib.AdamWOptions(
        0.0 if on_gpu[1] else float(lr), beta1, beta2, eps, weight_decay, max_norm,
        1 if on_gpu[0] else int(step),
        _one_value("step", step, torch.int64, first) if on_gpu[0] else None,
        _one_value("lr", lr, torch.float32, first) if on_gpu[1] else None,
        None if grad_norm is None else _one_value("grad_norm", grad_norm, torch.float32, first),
        int(seed) & 0xFFFFFFFF, 32 if wide else 8)
    # (host arrays of the library's types, which live until it has returned)
    at, sizes = array.array("Q", at), array.array("q", sizes[:n])

    def run():
        types_at = types.buffer_info()[0]
        hosts = [at.buffer_info()[0] + 8 * n * k for k in range(4 if wide else 6)] + [None] * (2 * wide)
        with _device(first):
            rc = _lib.load().mcx_adamw_step(*hosts, sizes.buffer_info()[0], types_at, types_at + 4 * n, n,
                                            options, _stream(first))
        _lib.check(rc, "adamw_step")
        _changed(lists[0] + every[2 * n:])
    return run


def adamw_moment(codes, scales, second, dtype=torch.float32):
    """The values of moments that adamw_step holds in 8 bits (`second`: the second ones), in
    codes' shape; float32 and bfloat16 hold them exactly."""
    _contig(codes=codes, scales=scales)
    _on_gpu("codes", codes, scales=scales)
    if codes.dtype != torch.uint8 or scales.dtype != torch.float32 or \
            scales.numel() != -(-codes.numel() // ADAMW_BLOCK):
        raise RuntimeError("codes must be uint8 and scales float32, one for %d of them" % ADAMW_BLOCK)
    if dtype not in _CLIP_DTYPES:
        raise RuntimeError("unsupported dtype %s (float32 or bfloat16)" % dtype)
    out = torch.empty(codes.shape, dtype=dtype, device=codes.device)
    with _device(codes):
        rc = _lib.load().mcx_adamw_moment(_ptr(codes), _ptr(scales), _ptr(out), codes.numel(),
                                          int(bool(second)), _CLIP_DTYPES[dtype], _stream(codes))
    _lib.check(rc, "adamw_moment")
    return out
