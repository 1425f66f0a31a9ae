"""ctypes binding of libsrgen.so (include/srgen.h).  The HIP library is the product path:
if it is missing this module raises -- there is no CPU or eager-PyTorch fallback."""
from __future__ import annotations

import ctypes
import os
import subprocess
import sys

_HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(_HERE, "csrc")
LIB_PATH = os.path.join(CSRC, "libsrgen.so")

SRGEN_F32, SRGEN_BF16, SRGEN_F16 = 0, 1, 2
NUM_TAPS = 11
DISC_NUM_TAPS = 10
TAP_NAMES = ("stem", "block0", "block7", "ca8", "block16", "ca17", "skip", "upsample", "output1",
             "ca8_scale", "ca17_scale")

KCLASS_NAMES = ("stem", "conv3x3_trunk", "conv3x3_up", "conv3x3_hr", "chan_attn", "head")

_lib = None


class SrgenError(RuntimeError):
    pass


class srgen_config(ctypes.Structure):
    _fields_ = [("num_blocks", ctypes.c_int32), ("in_ch", ctypes.c_int32), ("base_ch", ctypes.c_int32)]


class srdisc_config(ctypes.Structure):
    _fields_ = [("in_ch", ctypes.c_int32), ("base_ch", ctypes.c_int32)]


class srgen_moments(ctypes.Structure):
    _fields_ = [("bits", ctypes.c_int32), ("reserved", ctypes.c_int32), ("m", ctypes.c_void_p), ("v", ctypes.c_void_p),
                ("m_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p), ("step", ctypes.c_void_p),
                ("table", ctypes.c_void_p), ("numel", ctypes.c_uint64), ("chunks", ctypes.c_uint64)]


class srgen_adamw_args(ctypes.Structure):
    _fields_ = [("lr", ctypes.c_double), ("beta1", ctypes.c_double), ("beta2", ctypes.c_double), ("eps", ctypes.c_double),
                ("weight_decay", ctypes.c_double), ("lr_dev", ctypes.c_void_p), ("grad_mul", ctypes.c_void_p),
                ("grad_div", ctypes.c_void_p), ("found_inf", ctypes.c_void_p), ("norm_coef2", ctypes.c_void_p),
                ("norm_scratch", ctypes.c_void_p), ("norm_scratch_bytes", ctypes.c_size_t), ("max_norm", ctypes.c_double),
                ("seed", ctypes.c_uint32), ("maximize", ctypes.c_int32)]


def build(force: bool = False, jobs: int = 4) -> str:
    """Compile the gfx950 kernels + C ABI in-tree (hipcc cross-compiles without a GPU)."""
    cmd = ["make", "-C", CSRC, f"-j{jobs}", f"PYTHON={sys.executable}", "libsrgen.so", "../_tensorlist.so"]
    if force:
        cmd.insert(1, "-B")
    subprocess.check_call(cmd)
    return LIB_PATH


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise SrgenError(
            f"{LIB_PATH} is missing: the HIP extension is not built. Run "
            "`python -c 'import __graft_entry__ as g; g.build()'` (or `make -C superresolution_amd/csrc`). "
            "There is no fallback path.")
    L = ctypes.CDLL(LIB_PATH)
    vp, i, sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t
    L.srgen_abi_version.restype = i
    L.srgen_last_error.restype = ctypes.c_char_p
    L.srgen_create.argtypes = [ctypes.POINTER(srgen_config), ctypes.POINTER(vp)]
    L.srgen_destroy.argtypes = [vp]
    L.srgen_set_tensor.argtypes = [vp, ctypes.c_char_p, vp, sz]
    L.srgen_commit_weights.argtypes = [vp, vp]
    L.srgen_workspace_bytes.argtypes = [vp, i, i, ctypes.POINTER(sz)]
    L.srgen_forward.argtypes = [vp, vp, vp, vp, sz, i, i, vp]
    L.srgen_forward_train.argtypes = [vp, vp, vp, vp, sz, i, vp, vp]
    L.srgen_forward_train.restype = i
    L.srgen_forward_taps.argtypes = [vp, vp, vp, vp, sz, i, i, ctypes.POINTER(vp), vp]
    L.srgen_forward_profile.argtypes = [vp, vp, vp, vp, sz, i, i, vp, ctypes.POINTER(ctypes.c_float),
                                        ctypes.POINTER(ctypes.c_int)]
    L.srgen_bilinear_resize.argtypes = [vp, vp, i, i, i, i, i, vp]
    L.srgen_normalize.argtypes = [vp, vp, sz, ctypes.c_float, i, vp]
    L.srgen_metrics_scratch_bytes.argtypes = [i, i, i, i, ctypes.POINTER(sz)]
    L.srgen_metrics.argtypes = [vp, vp, i, i, i, i, vp, vp, sz, vp]
    L.srgen_metrics_noalloc.argtypes = [vp, vp, i, i, i, i, vp, vp]
    L.srgen_metrics_noalloc.restype = i
    L.srgen_pixel_losses.argtypes = [vp, vp, i, i, i, i, vp, vp, sz, vp]
    L.srgen_pixel_losses.restype = i
    L.srdisc_create.argtypes = [ctypes.POINTER(srdisc_config), ctypes.POINTER(vp)]
    L.srdisc_destroy.argtypes = [vp]
    L.srdisc_set_tensor.argtypes = [vp, ctypes.c_char_p, vp, sz]
    L.srdisc_commit_weights.argtypes = [vp, vp]
    L.srdisc_workspace_bytes.argtypes = [vp, i, i, i, ctypes.POINTER(sz)]
    L.srdisc_forward.argtypes = [vp, vp, vp, vp, sz, i, i, i, ctypes.POINTER(vp), vp]
    L.srgen_ragan_loss.argtypes = [vp, vp, sz, sz, ctypes.c_float, ctypes.c_float, vp, vp]
    f = ctypes.c_float
    L.srgen_wino_pack.argtypes = [vp, i, i, i, vp, vp]
    L.srgen_conv3x3_nhwc.argtypes = [vp, vp, vp, vp, vp, i, i, i, i, vp]
    L.srgen_split_pack.argtypes = [vp, i, i, i, vp, vp]
    L.srgen_split_pack_many.argtypes = [i, ctypes.POINTER(vp), ctypes.POINTER(i), ctypes.POINTER(i), ctypes.POINTER(i),
                                        ctypes.POINTER(vp), vp]
    L.srgen_conv3x3_nhwc_split.argtypes = [vp, vp, vp, vp, vp, i, i, i, i, vp, vp]
    L.srgen_conv3x3_nhwc_f16.argtypes = [vp, vp, vp, vp, vp, i, i, i, i, vp, vp]
    L.srgen_absmax.argtypes = [vp, sz, vp, vp]
    L.srgen_conv3x3_wgrad_scratch_bytes.argtypes = [i, i, ctypes.POINTER(sz)]
    L.srgen_conv3x3_wgrad.argtypes = [vp, vp, i, i, vp, vp, vp, sz, vp]
    L.srgen_conv3x3_wgrad_split.argtypes = [vp, vp, i, i, vp, vp, vp, vp, sz, vp]
    L.srgen_conv3x3_wgrad_f16.argtypes = [vp, vp, i, i, vp, vp, vp, vp, sz, vp]
    L.srgen_bn_train_scratch_bytes.argtypes = [ctypes.POINTER(sz)]
    L.srgen_bn_train_fwd.argtypes = [vp, vp, vp, vp, vp, vp, f, vp, sz, vp, sz, vp]
    L.srgen_bn_train_bwd.argtypes = [vp, vp, vp, vp, vp, vp, f, vp, vp, vp, vp, sz, vp, sz, vp, vp]
    L.srgen_pixel_loss_grad.argtypes = [vp, vp, i, i, i, i, f, f, vp, vp, sz, vp]
    L.srgen_adamw.argtypes = [vp, vp, vp, vp, sz, f, f, f, f, f, i, vp]
    L.srgen_prelu_scratch_bytes.argtypes = [ctypes.POINTER(sz)]
    L.srgen_prelu_scalar_fwd.argtypes = [vp, vp, vp, sz, vp]
    L.srgen_prelu_scalar_bwd.argtypes = [vp, vp, vp, vp, vp, vp, sz, vp, sz, vp]
    L.srgen_prelu_scalar_bwd_unshuffle.argtypes = [vp, vp, vp, vp, vp, i, i, vp, sz, vp]
    L.srgen_prelu_scalar_bwd_unshuffle.restype = i
    L.srgen_prelu_scalar_bwd_unshuffle_bf16.argtypes = L.srgen_prelu_scalar_bwd_unshuffle.argtypes
    L.srgen_prelu_scalar_bwd_unshuffle_bf16.restype = i
    L.srgen_conv9x9_c3_nhwc.argtypes = [vp, vp, vp, vp, i, i, i, i, i, i, vp]
    L.srgen_conv9x9_c3_nhwc_split.argtypes = [vp, vp, vp, vp, i, i, i, i, i, i, vp, sz, vp]
    L.srgen_conv9x9_c3_wgrad_scratch_bytes.argtypes = [i, i, ctypes.POINTER(sz)]
    L.srgen_conv9x9_c3_wgrad.argtypes = [vp, vp, i, i, i, i, i, i, vp, vp, vp, sz, vp]
    L.srgen_head_nhwc.argtypes = [vp, vp, vp, vp, i, vp]
    L.srgen_head_nhwc_split.argtypes = [vp, vp, vp, vp, i, vp]
    L.srgen_chan_attn_nhwc.argtypes = [vp, vp, vp, vp, vp, vp, vp, i, vp]
    L.srgen_chan_attn_bwd_scratch_bytes.argtypes = [i, ctypes.POINTER(sz)]
    L.srgen_chan_attn_bwd.argtypes = [vp, vp, vp, vp, i, vp, vp, vp, vp, vp, vp, vp, vp, vp, vp, sz, vp]
    # the 16-bit step (bf16 activation / gradient tensors)
    L.srgen_bf16_pack_many.argtypes = L.srgen_split_pack_many.argtypes
    L.srgen_conv3x3_nhwc_bf16.argtypes = [vp, vp, vp, vp, vp, i, i, i, i, vp]
    L.srgen_conv3x3_wgrad_bf16.argtypes = [vp, vp, i, i, vp, vp, vp, sz, vp]
    L.srgen_bn_train_fwd_bf16.argtypes = L.srgen_bn_train_fwd.argtypes
    L.srgen_bn_train_bwd_bf16.argtypes = [vp, vp, vp, vp, vp, vp, f, vp, vp, vp, vp, sz, vp, sz, vp]
    L.srgen_prelu_scalar_fwd_bf16.argtypes = L.srgen_prelu_scalar_fwd.argtypes
    L.srgen_prelu_scalar_bwd_bf16.argtypes = L.srgen_prelu_scalar_bwd.argtypes
    L.srgen_conv9x9_c3_nhwc_split_bf16.argtypes = L.srgen_conv9x9_c3_nhwc_split.argtypes
    L.srgen_conv9x9_c3_wgrad_bf16.argtypes = L.srgen_conv9x9_c3_wgrad.argtypes
    L.srgen_head_nhwc_bf16.argtypes = L.srgen_head_nhwc.argtypes
    L.srgen_chan_attn_nhwc_bf16.argtypes = L.srgen_chan_attn_nhwc.argtypes
    L.srgen_chan_attn_bwd_bf16.argtypes = L.srgen_chan_attn_bwd.argtypes
    for name in ("srgen_bf16_pack_many", "srgen_conv3x3_nhwc_bf16", "srgen_conv3x3_wgrad_bf16", "srgen_bn_train_fwd_bf16",
                 "srgen_bn_train_bwd_bf16", "srgen_prelu_scalar_fwd_bf16", "srgen_prelu_scalar_bwd_bf16",
                 "srgen_conv9x9_c3_nhwc_split_bf16", "srgen_conv9x9_c3_wgrad_bf16", "srgen_head_nhwc_bf16",
                 "srgen_chan_attn_nhwc_bf16", "srgen_chan_attn_bwd_bf16"):
        getattr(L, name).restype = i
    psz = ctypes.POINTER(sz)
    L.srdisc_pack.argtypes = [vp, i, i, i, vp, vp]
    L.srdisc_stem_nhwc.argtypes = [vp, vp, vp, vp, i, i, i, f, vp]
    L.srdisc_conv_nhwc.argtypes = [vp, vp, vp, vp, vp, i, i, i, i, i, i, f, vp]
    L.srdisc_tail.argtypes = [vp, vp, vp, vp, i, i, i, i, vp]
    L.srdisc_conv_dgrad2.argtypes = [vp, vp, vp, vp, i, i, i, i, i, f, vp]
    L.srdisc_conv_dgrad2.restype = i
    L.srdisc_conv_wgrad_scratch_bytes.argtypes = [i, i, i, i, i, psz]
    L.srdisc_conv_wgrad.argtypes = [vp, vp, i, i, i, i, i, i, vp, vp, vp, sz, vp]
    L.srdisc_conv_wgrad_bf16p.argtypes = L.srdisc_conv_wgrad.argtypes
    L.srdisc_conv_wgrad_bf16p.restype = i
    L.srdisc_stem_wgrad_scratch_bytes.argtypes = [psz]
    L.srdisc_stem_wgrad.argtypes = [vp, vp, i, i, i, vp, vp, vp, sz, vp]
    L.srdisc_stem_dgrad.argtypes = [vp, vp, i, i, i, vp, vp]
    L.srdisc_tail_bwd.argtypes = [vp, vp, vp, i, i, i, i, f, vp, vp, vp, vp]
    L.srgen_ragan_loss_grad.argtypes = [vp, vp, sz, sz, f, f, f, vp, vp, vp]
    L.srdisc_pack_bf16.argtypes = L.srdisc_pack.argtypes
    L.srdisc_conv_nhwc_bf16p.argtypes = L.srdisc_conv_nhwc.argtypes
    L.srdisc_conv_dgrad2_bf16p.argtypes = L.srdisc_conv_dgrad2.argtypes
    for name in ("srdisc_pack_bf16", "srdisc_conv_nhwc_bf16p", "srdisc_conv_dgrad2_bf16p"):
        getattr(L, name).restype = i
    L.srgen_clip_grad_norm_scratch_bytes.argtypes = [psz]
    L.srgen_clip_grad_norm.argtypes = [vp, sz, f, vp, vp, sz, vp]
    for name in ("srdisc_pack", "srdisc_stem_nhwc", "srdisc_conv_nhwc", "srdisc_tail",
                 "srdisc_conv_wgrad_scratch_bytes", "srdisc_conv_wgrad", "srdisc_stem_wgrad_scratch_bytes", "srdisc_stem_wgrad",
                 "srdisc_stem_dgrad", "srdisc_tail_bwd", "srgen_ragan_loss_grad", "srgen_clip_grad_norm_scratch_bytes",
                 "srgen_clip_grad_norm"):
        getattr(L, name).restype = i
    for name in ("srgen_prelu_scratch_bytes", "srgen_prelu_scalar_fwd", "srgen_prelu_scalar_bwd", "srgen_conv9x9_c3_nhwc", "srgen_conv9x9_c3_nhwc_split",
                 "srgen_conv9x9_c3_wgrad_scratch_bytes", "srgen_conv9x9_c3_wgrad", "srgen_head_nhwc", "srgen_head_nhwc_split", "srgen_chan_attn_nhwc",
                 "srgen_chan_attn_bwd_scratch_bytes", "srgen_chan_attn_bwd"):
        getattr(L, name).restype = i
    for name in ("srgen_split_pack_many", "srgen_conv3x3_nhwc_f16", "srgen_conv3x3_wgrad_f16", "srgen_wino_pack", "srgen_conv3x3_nhwc", "srgen_split_pack", "srgen_conv3x3_nhwc_split", "srgen_absmax", "srgen_conv3x3_wgrad_scratch_bytes", "srgen_conv3x3_wgrad", "srgen_conv3x3_wgrad_split",
                 "srgen_bn_train_scratch_bytes", "srgen_bn_train_fwd", "srgen_bn_train_bwd", "srgen_pixel_loss_grad",
                 "srgen_adamw"):
        getattr(L, name).restype = i
    for name in ("srdisc_create", "srdisc_destroy", "srdisc_set_tensor", "srdisc_commit_weights",
                 "srdisc_workspace_bytes", "srdisc_forward", "srgen_ragan_loss"):
        getattr(L, name).restype = i
    for name in ("srgen_create", "srgen_destroy", "srgen_set_tensor", "srgen_commit_weights",
                 "srgen_workspace_bytes", "srgen_forward", "srgen_forward_taps", "srgen_forward_profile", "srgen_bilinear_resize", "srgen_normalize",
                 "srgen_metrics_scratch_bytes", "srgen_metrics"):
        getattr(L, name).restype = i
    L.srgen_adamw_chunk_count.argtypes = [i, vp, ctypes.POINTER(ctypes.c_uint64)]
    L.srgen_adamw_chunk_table.argtypes = [i, vp, vp, vp, ctypes.c_uint64]
    L.srgen_adamw_many.argtypes = [i, vp, vp, vp, vp, vp, vp, ctypes.POINTER(srgen_moments), ctypes.POINTER(srgen_adamw_args), vp]
    L.srgen_total_norm_scratch_bytes.argtypes = [i, vp, psz]
    L.srgen_total_norm.argtypes = [i, vp, vp, vp, ctypes.c_double, vp, vp, sz, vp]
    L.srgen_scale_many.argtypes = [i, vp, vp, vp, vp, vp]
    L.srgen_moments_pack.argtypes = [vp, vp, sz, vp, vp, vp, vp, vp]
    L.srgen_moments_unpack.argtypes = [vp, vp, vp, vp, vp, vp, sz, vp]
    for name in ("srgen_adamw_chunk_count", "srgen_adamw_chunk_table", "srgen_adamw_many", "srgen_total_norm_scratch_bytes", "srgen_total_norm",
                 "srgen_scale_many", "srgen_moments_pack", "srgen_moments_unpack"):
        getattr(L, name).restype = i
    if L.srgen_abi_version() != 1:
        raise SrgenError(f"libsrgen.so ABI version {L.srgen_abi_version()} != 1; rebuild it")
    _lib = L
    return L


def check(rc: int, module: str = "Generator") -> None:
    """Map a negative srgen return code to a Python exception carrying srgen_last_error()."""
    if rc == 0:
        return
    msg = lib().srgen_last_error().decode("utf-8", "replace")
    if rc == -2:                       # SRGEN_E_KEY: same exception type load_state_dict raises
        raise RuntimeError(f"Error(s) in loading state_dict for {module}: {msg}")
    raise SrgenError(f"libsrgen error {rc}: {msg}")
