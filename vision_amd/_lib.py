"""ctypes binding of libvision_amd.so (the C ABI declared in include/vision_amd.h).

The library is built in-tree by `python vision_amd/build_ext.py` (hipcc, gfx950).  There is no
fallback: if the shared object is missing, importing this module raises.
"""
import ctypes as C
import os

# torch must be imported first: its wheel bundles the HIP runtime (libamdhip64) that owns the
# device memory and streams handed to this library; loading libvision_amd.so first would pull a
# second copy of the runtime from /opt/rocm into the process.
import torch  # noqa: F401
from torch.autograd import forward_ad

_HERE = os.path.dirname(os.path.abspath(__file__))
# VAMD_LIB: another build of the same library (side-by-side kernel experiments)
LIB_PATH = os.environ.get("VAMD_LIB") or os.path.join(_HERE, "lib", "libvision_amd.so")

F32, BF16 = 0, 1
KV_E4M3, KV_INT8 = 0, 1
ALGO_AUTO, ALGO_DIRECT, ALGO_MFMA, ALGO_THIN = 0, 1, 2, 3


class VamdError(RuntimeError):
    pass


_DEFAULT_SCRATCH = None      # (tensor, nbytes) attached to every new ConvDesc (set_default_scratch)


class ConvDesc(C.Structure):
    _fields_ = [(n, C.c_int32) for n in
                ("B", "H", "W", "Cin", "Cout", "ksize", "stride", "pad", "upsample", "dtype", "algo")] + \
               [("scratch", C.c_void_p), ("scratch_bytes", C.c_uint64)]

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        if _DEFAULT_SCRATCH is not None and not self.scratch:
            self.scratch, self.scratch_bytes = _DEFAULT_SCRATCH[0].data_ptr(), _DEFAULT_SCRATCH[1]


def set_default_scratch(tensor):
    """Attach `tensor` (zero-filled uint8 device memory of CONV_SCRATCH_BYTES, or None) to every ConvDesc created
    from now on that names no scratch buffer of its own (tests and micro-benchmarks; the engine passes its own)."""
    global _DEFAULT_SCRATCH
    _DEFAULT_SCRATCH = None if tensor is None else (tensor, tensor.numel() * tensor.element_size())


CONV_SCRATCH_BYTES = 4096 + 256 * 256 * 256 * 4      # VAMD_CONV_SCRATCH_BYTES


class RepackItem(C.Structure):
    _fields_ = [("w", C.c_void_p), ("w_fwd", C.c_void_p), ("w_dgrad", C.c_void_p), ("first_block", C.c_longlong),
                ("Cout", C.c_int32), ("Cin", C.c_int32), ("ksize", C.c_int32), ("ld_dgrad", C.c_int32),
                ("bias", C.c_void_p), ("bias_out", C.c_void_p), ("w_up4_dgrad", C.c_void_p), ("w_up4_fwd", C.c_void_p)]


class LinearItem(C.Structure):
    _fields_ = [("W", C.c_void_p), ("bias", C.c_void_p), ("y", C.c_void_p), ("O", C.c_int32), ("first", C.c_int32)]


class LinearBwdItem(C.Structure):
    _fields_ = [("W", C.c_void_p), ("dy", C.c_void_p), ("dW", C.c_void_p), ("dbias", C.c_void_p), ("O", C.c_int32),
                ("pad_", C.c_int32)]


if not os.path.exists(LIB_PATH):
    raise ImportError(
        f"{LIB_PATH} not found: build the HIP extension first (python vision_amd/build_ext.py). "
        "vision_amd has no CPU or eager fallback.")

lib = C.CDLL(LIB_PATH)

_p, _i, _l, _f, _z = C.c_void_p, C.c_int, C.c_int64, C.c_float, C.c_size_t
_d = C.POINTER(ConvDesc)

# name -> (restype, argtypes); mirrors include/vision_amd.h one to one
SIGNATURES = {
    "vamd_last_error": (C.c_char_p, []),
    "vamd_version": (_i, []),
    "vamd_launch_timing": (_i, [_i]),
    "vamd_launch_timing_read": (C.c_long, [_i, C.POINTER(C.c_double), C.POINTER(C.c_double), C.POINTER(C.c_double)]),
    "vamd_conv2d_fwd": (_i, [_d, _p, _p, _p, _p, _p, _p, _p, _p]),
    "vamd_conv2d_fwd_stats": (_i, [_d, _p, _p, _p, _p, _p, _p, _p, _p, _p]),
    "vamd_conv2d_fwd_act_supported": (_i, [_d]),
    "vamd_conv2d_fwd_act": (_i, [_d, _p, _p, _p, _p, _p, _p, _p, _p, _f, _p, _p, _p]),
    "vamd_conv2d_stats_parts": (_i, [_d]),
    "vamd_conv2d_fwd_short_supported": (_i, [_d, _i]),
    "vamd_conv2d_fwd_short": (_i, [_d, _p, _p, _p, _p, _p, _p, _i, _p, _p, _p, _p]),
    "vamd_fold_partials": (_i, [_p, _i, _i, _i, _p, _p]),
    "vamd_conv2d_dgrad": (_i, [_d, _p, _p, _p, _p, _p, _z, _p]),
    "vamd_conv2d_dgrad_workspace": (_z, [_d]),
    "vamd_conv2d_fwd_up4_supported": (_i, [_d]),
    "vamd_conv2d_fwd_up4_stats_parts": (_i, [_d]),
    "vamd_conv2d_fwd_up4": (_i, [_d, _p, _p, _p, _p, _p, _p, _p, _p, _p]),
    "vamd_repack_weight_up4_fwd": (_i, [_p, _p, _i, _i, _i, _p]),
    "vamd_conv2d_dgrad_up4_supported": (_i, [_d]),
    "vamd_conv2d_dgrad_up4": (_i, [_d, _p, _p, _p, _p, _p]),
    "vamd_repack_weight_up4": (_i, [_p, _p, _i, _i, _i, _p]),
    "vamd_conv2d_wgrad": (_i, [_d, _p, _p, _p, _p, _p, _z, _p]),
    "vamd_conv2d_wgrad_oihw": (_i, [_d, _p, _p, _p, _p, _p, _z, _p]),
    "vamd_conv2d_wgrad_workspace": (_z, [_d]),
    "vamd_conv2d_wgrad_oihw_split3": (_i, [_d, _p, _p, C.POINTER(C.c_void_p * 3), C.POINTER(C.c_void_p * 3), _p, _z, _p]),
    "vamd_conv2d_prenorm_supported": (_i, [_d]),
    "vamd_conv2d_fwd_prenorm": (_i, [_d, _p, _p, _p, _f, _p, _p, _p, _p, _p, _p, _p, _p]),
    "vamd_conv2d_wgrad_prenorm_oihw": (_i, [_d, _p, _p, _p, _p, _f, _p, _p, _p, _z, _p]),
    "vamd_conv_splitk": (_i, [_i]),
    "vamd_conv2d_uses_mfma": (_i, [_d, _i]),
    "vamd_repack_weight": (_i, [_p, _p, _p, _i, _i, _i, _i, _p]),
    "vamd_repack_weights": (_i, [_p, _i, C.c_longlong, _i, _p]),
    "vamd_unpack_wgrad": (_i, [_p, _p, _i, _i, _i, _p]),
    "vamd_stats_chunks": (_i, [_l, _i]),
    "vamd_stream_wait": (_i, [_p, _p]),
    "vamd_chan_stats": (_i, [_p, _p, _i, _l, _i, _i, _p]),
    "vamd_norm_bwd_stats": (_i, [_p, _p, _p, _p, _p, _p, _p, _f, _f, _p, _i, _l, _i, _i, _p]),
    "vamd_bn_finalize": (_i, [_p, _i, _i, _l, _p, _p, _p, _p, _p, _f, _f, _i, _p, _p, _p, _p, _p]),
    "vamd_gn_finalize": (_i, [_p, _i, _i, _i, _i, _l, _p, _p, _f, _p, _p, _p, _p, _p]),
    "vamd_gn_coef_noalloc": (_i, [_p, _i, _i, _i, _l, _p, _p, _f, _p, _p, _p, _p, _i, _p]),
    "vamd_scale_shift_act": (_i, [_p, _p, _p, _p, _f, _f, _p, _i, _l, _i, _i, _p]),
    "vamd_bn_bwd_finalize": (_i, [_p, _i, _i, _l, _p, _p, _p, _p, _p, _p, _i, _p]),
    "vamd_bn_bwd_stats_img": (_i, [_p, _p, _p, _p, _p, _p, _p, _f, _f, _p, _i, _l, _i, _i, _p]),
    "vamd_bn_bwd_finalize_img": (_i, [_p, _i, _i, _i, _l, _p, _p, _p, _p, _p, _p, _p, _p, _i, _p]),
    "vamd_gn_bwd_finalize": (_i, [_p, _i, _i, _i, _i, _l, _p, _p, _p, _p, _p, _p, _p, _p]),
    "vamd_norm_bwd_apply": (_i, [_p, _p, _p, _p, _p, _p, _p, _f, _f, _p, _p, _p, _p, _p, _p, _i, _l, _i, _i, _p]),
    "vamd_sum_finalize": (_i, [_p, _i, _i, _i, _p, _p, _p]),
    "vamd_bmm_nt": (_i, [_p, _p, _p, _i, _i, _i, _i, _i, _i, _i, _f, _i, _i, _i, _p]),
    "vamd_bmm_tn": (_i, [_p, _p, _p, _i, _i, _i, _i, _i, _i, _i, _f, _i, _i, _p]),
    "vamd_sumpool2x2": (_i, [_p, _p, _i, _i, _i, _i, _i, _p]),
    "vamd_pool2x2": (_i, [_p, _p, _p, _i, _i, _i, _i, _f, _i, _p]),
    "vamd_unpool2x2": (_i, [_p, _p, _p, _i, _i, _i, _i, _i, _i, _f, _i, _p]),
    "vamd_transpose": (_i, [_p, _p, _i, _i, _i, _i, _i, _p]),
    "vamd_transpose_ld": (_i, [_p, _p, _i, _i, _i, _i, _i, _i, _p]),
    "vamd_attention_fwd_supported": (_i, [_i, _i, _i]),
    "vamd_attention_fwd": (_i, [_p, _p, _p, _p, _i, _i, _i, _i, _f, _i, _p]),
    "vamd_softmax_rows": (_i, [_p, _p, _l, _i, _i, _i, _p]),
    "vamd_softmax_rows_bwd": (_i, [_p, _p, _p, _l, _i, _i, _f, _i, _p]),
    "vamd_add": (_i, [_p, _p, _p, _l, _i, _p]),
    "vamd_timeembed": (_i, [_p, _p, _p, _i, _i, _p]),
    "vamd_linear_fwd": (_i, [_p, _p, _p, _p, _i, _i, _i, _i, _f, _p]),
    "vamd_linear_fwd_multi": (_i, [_p, _p, _i, _i, _i, _i, _i, _f, _p]),
    "vamd_linear_bwd_multi": (_i, [_p, _p, _i, _i, _i, _i, _i, _f, _p, _i, _p]),
    "vamd_linear_bwd": (_i, [_p, _p, _p, _p, _p, _p, _i, _i, _i, _i, _f, _i, _p]),
    "vamd_qsample": (_i, [_p, _p, _p, _p, _p, _p, _p, _i, _i, _i, _i, _i, _p]),
    "vamd_schedule": (_i, [_p, _p, _p, _p, _i, _p]),
    "vamd_l1_chunks": (_i, [_l]),
    "vamd_l1_loss_fwd": (_i, [_p, _p, _p, _p, _i, _i, _i, _i, _i, _p]),
    "vamd_l1_loss_bwd": (_i, [_p, _p, _p, _p, _i, _i, _i, _i, _i, _p]),
    "vamd_denoise_step": (_i, [_p, _p, _p, _p, _p, _p, _p, _p, _i, _i, _i, _i, _i, _p]),
    "vamd_nchw_to_nhwc": (_i, [_p, _p, _p, _i, _i, _i, _i, _i, _p]),
    "vamd_nhwc_to_nchw": (_i, [_p, _p, _i, _i, _i, _i, _i, _p]),
    "vamd_adamw": (_i, [_p, _p, _p, _p, _l, _f, _p, _f, _f, _f, _f, _i, _f, _p]),
    "vamd_adam_l2": (_i, [_p, _p, _p, _p, _l, _f, _p, _f, _f, _f, _f, _i, _f, _p]),
    "vamd_adam_dev": (_i, [_p, _p, _p, _p, _l, _p, _p, _f, _f, _f, _f, _f, _i, _p]),
    "vamd_resize_ksize": (_i, [_i, _i]),
    "vamd_resize_coeffs": (_i, [_i, _i, _p, _p, _i]),
    "vamd_image_resize_u8": (_i, [_p, _i, _i, _i, _p, _p, _i, _p, _p, _i, _p, _i, _i, _p, _p, _p]),
    "vamd_add_cast": (_i, [_p, _i, _p, _i, _p, _i, _l, _p]),
    "vamd_sigmoid_mse_fwd": (_i, [_p, _p, _p, _p, _p, _i, _i, _i, _i, _i, _p]),
    "vamd_sigmoid_mse_bwd": (_i, [_p, _p, _p, _p, _p, _i, _i, _i, _i, _i, _p]),
    "vamd_vq_workspace": (_z, [_l]),
    "vamd_vq_forward": (_i, [_p, _p, _l, _i, _i, _i, _i, _f, _p, _p, _p, _p, _z, _p]),
    "vamd_vq_backward": (_i, [_p, _p, _p, _p, _p, _l, _i, _i, _i, _i, _f, _p, _p, _p]),
    "vamd_rotary": (_i, [_p, _i, _p, _f, _l, _l, _i, _i, _i, _i] + [_p, _p, _i, _l, _l, _l, _l, _l, _l] * 2 + [_i, _p]),
    "vamd_kv_append": (_i, [_p, _l, _l, _p, _l, _l, _p, _p, _p, _p, _p, _l, _p, _p, _l] + [_i] * 9 + [_p]),
    "vamd_kv_read": (_i, [_p, _p, _p, _p, _p, _l, _p, _p, _l] + [_i] * 8 + [_p, _l, _l, _p, _l, _l, _i, _p]),
    "vamd_kv_attend_tile": (_i, [_l, _i, _i, _l, _i, _i, _i, _i, _i, _i]),
    "vamd_kv_attend_workspace": (_z, [_l, _i, _i, _l, _i, _i, _i, _i, _i, _i]),
    "vamd_kv_attend": (_i, [_p, _l, _l, _p, _p, _p, _p, _p, _l, _p, _p, _l, _i, _i, _l] + [_i] * 7 +
                       [_f, _i, _i, _i, _p, _l, _l, _p, _z, _i, _p]),
}

for _name, (_res, _args) in SIGNATURES.items():
    _fn = getattr(lib, _name)          # AttributeError here = header and library out of sync
    _fn.restype = _res
    _fn.argtypes = _args


def source_hash():
    """sha256 over the kernel sources and the header: profile summaries are stamped with it, so a reader can
    tell whether a committed counter pass still describes the kernels in the tree."""
    import hashlib
    h = hashlib.sha256()
    csrc = os.path.join(_HERE, "csrc")
    for f in sorted(os.listdir(csrc)) + [os.path.join(_HERE, "..", "include", "vision_amd.h")]:
        with open(f if os.path.isabs(f) or f.startswith(_HERE) else os.path.join(csrc, f), "rb") as fh:
            h.update(fh.read())
    return h.hexdigest()[:16]


def check(rc, what=""):
    if rc != 0:
        msg = lib.vamd_last_error().decode(errors="replace")
        raise VamdError(f"{what or 'libvision_amd'} failed (status {rc}): {msg}")


def call(name, *args):
    """Call an int-returning entry point and raise VamdError on a non-zero status."""
    check(getattr(lib, name)(*args), name)


_PROXY = torch._C._TorchDispatchModeKey.PROXY
_tracing, _modes, _functions = torch._C._get_tracing_state, torch._C._len_torch_dispatch_stack, torch._C._len_torch_function_stack
_before_dispatch = torch._ops.mode_stack_state_for_pre_dispatch()
_entries = {name: getattr(lib, name) for name in SIGNATURES}


def call_on(device, name, *args):
    """The same on the current stream of `device` (its last argument), whichever device is current.  A kernel launched from here is
    invisible to what records torch's operators, whose program would return memory that nobody writes: refused there."""
    if _tracing() is not None or (_modes() and torch._C._get_dispatch_mode(_PROXY) is not None) or (_functions() and _before_dispatch.count()):
        raise RuntimeError(f"{name} cannot be recorded by torch.jit.trace or make_fx: call it outside of the traced function")
    index = device.index
    if index == torch.cuda.current_device():
        rc = _entries[name](*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = _entries[name](*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        check(rc, name)


def overwritten(*tensors):
    """Tells autograd that a kernel writes into these tensors (None: no tensor): a backward pass that has saved one of them refuses to run."""
    for t in tensors:
        if t is not None and t.numel() and not t.is_inference():
            torch.autograd.graph.increment_version(t)


def has_tangent(t):
    """Whether t is a dual number of forward-mode differentiation (whether or not it requires a gradient)."""
    return forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None


def self_overlapping(t):
    """Whether two elements of t may share memory (as those of an expanded tensor do)."""
    reach = 0
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride <= reach:
            return True
        reach += stride * (size - 1)
    return False


def overlapping(a, b):
    """Whether some element of a shares memory with one of b (tensors of one element size on one device): exact, also for pieces of one
    buffer's rows, and whatever storages they belong to.

    Elements meet where sum(i * stride of a) - sum(j * stride of b) is the distance of the two; largest strides first, few
    multiples of each leave a rest that the smaller ones can make up."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    u, v = a.untyped_storage(), b.untyped_storage()
    at, to = u.data_ptr(), v.data_ptr()
    if at != to and (at + u.nbytes() <= to or to + v.nbytes() <= at):
        return False                                    # no memory in common, whatever of it they use
    size = a.element_size()
    ahead = b.data_ptr() - a.data_ptr()                 # (addresses: tensors of different storages may lie in the same memory)
    u, v = a.stride(), b.stride()
    if len(u) == len(v) > 2 and u[:-2] == v[:-2] and u[-3] > 0 and ahead % size == 0 and all(s % u[-3] == 0 for s in u[:-3]):
        # side by side in the rows of one buffer (queries and keys of one projection): told without what follows
        at = ahead // size % u[-3]
        if at > (a.shape[-2] - 1) * u[-2] + (a.shape[-1] - 1) * u[-1] and u[-3] - at > (b.shape[-2] - 1) * v[-2] + (b.shape[-1] - 1) * v[-1]:
            return False
    ranges = {}                                         # stride -> [least, most] multiple
    for t, end, sign in ((a, 1, 1), (b, 0, -1)):
        for n, s in zip(t.shape, t.stride()):
            if n > 1 and s:
                ranges.setdefault(s, [0, 0])[end] += sign * (n - 1)
    low, high = sum(s * r[0] for s, r in ranges.items()), sum(s * r[1] for s, r in ranges.items())
    if not (low - 1) * size < ahead < (high + 1) * size:
        return False
    if ahead % size:
        return True                                     # (elements may meet in part: not looked at more closely)
    rests = {ahead // size}
    for s in sorted(ranges, reverse=True):
        least, most = ranges[s]
        low, high = low - s * least, high - s * most    # what the smaller strides can add
        rests = {rest - d * s for rest in rests for d in range(max(least, -((high - rest) // s)), min(most, (rest - low) // s) + 1)}
        if len(rests) > 4096:
            return True
    return 0 in rests
