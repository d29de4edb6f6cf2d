"""ctypes binding of libsaunet_hip.so (C ABI declared in include/saunet_hip.h).

There is NO fallback: if the HIP library cannot be loaded every op raises.  Each wrapper takes
torch tensors only for their ``data_ptr()`` / shape; torch is plumbing (memory + streams).
"""
import ctypes as C
import os

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("SAUNET_HIP_LIB") or os.path.join(_HERE, "libsaunet_hip.so")      # the override serves A/B kernel measurements

F32, BF16, F16 = 0, 1, 2
PACK_FWD, PACK_DGRAD, PACK_CONVT_FWD, PACK_CONVT_DGRAD = 0, 1, 2, 3


class ConvDesc(C.Structure):
    _fields_ = [(n, C.c_int32) for n in (
        "dtype", "N", "H", "W", "Cin", "ldx", "Ho", "Wo", "Cout", "ldy", "KH", "KW", "stride", "pad",
        "transposed", "pro_relu", "stat_replicas", "stat_rstride", "epi_relu")] + [("workspace", C.c_void_p), ("workspace_bytes", C.c_int64)]


class BnEpilogue(C.Structure):
    _fields_ = [("bn_x", C.c_void_p), ("ld_bn_x", C.c_int32), ("relu", C.c_int32), ("accumulate", C.c_int32), ("reserved", C.c_int32),
                ("scale", C.c_void_p), ("shift", C.c_void_p),
                ("mean", C.c_void_p), ("invstd", C.c_void_p), ("sums", C.c_void_p), ("sums_replicas", C.c_int32), ("sums_rstride", C.c_int32),
                ("relu_mask", C.c_void_p)]


class BnPrologue(C.Structure):
    _fields_ = [("sum", C.c_void_p), ("sumsq", C.c_void_p), ("replicas", C.c_int32), ("rstride", C.c_int32), ("count", C.c_double),
                ("eps", C.c_float), ("momentum", C.c_float), ("c_lo", C.c_int32), ("ld_xhat", C.c_int32), ("xhat", C.c_void_p),
                ("gamma", C.c_void_p), ("beta", C.c_void_p), ("params", C.c_void_p), ("running_mean", C.c_void_p), ("running_var", C.c_void_p)]


class PackList(C.Structure):
    _fields_ = [("count", C.c_int32), ("mode", C.c_int32 * 64), ("dims", (C.c_int32 * 4) * 64), ("src", C.c_void_p * 64),
                ("dst", C.c_void_p * 64)]


WGRAD_REDUCE_MAX = 64


class WgradPending(C.Structure):
    _fields_ = [("ws", C.c_void_p), ("dw", C.c_void_p), ("wsize", C.c_int64), ("groups", C.c_int32), ("taps", C.c_int32)]


class WgradReduceList(C.Structure):
    _fields_ = [("count", C.c_int32), ("reserved", C.c_int32), ("item", WgradPending * WGRAD_REDUCE_MAX)]


WGRAD_GROUP_MAX = 32


class WgradGroupItem(C.Structure):
    _fields_ = [("x", C.c_void_p), ("dy", C.c_void_p), ("dw", C.c_void_p), ("pro_scale", C.c_void_p), ("pro_shift", C.c_void_p),
                ("Cin", C.c_int32), ("ldx", C.c_int32), ("Cout", C.c_int32), ("lddy", C.c_int32)]


class WgradGroup(C.Structure):
    _fields_ = [(n, C.c_int32) for n in "dtype N H W KH pad pro_relu count".split()] + [("item", WgradGroupItem * WGRAD_GROUP_MAX)]


class DenseLayerBwd(C.Structure):
    """saunet_dense_layer_bwd"""
    _fields_ = [(n, C.c_int32) for n in "N H W Cin Ctot c_begin".split()] + [
        ("buf", C.c_void_p), ("dbuf", C.c_void_p), ("xhat", C.c_void_p), ("ld_xhat", C.c_int32), ("reserved2", C.c_int32),
        ("ab", C.c_void_p), ("ab_replicas", C.c_int32), ("ab_rstride", C.c_int32), ("count", C.c_double),
        ("z1", C.c_void_p), ("g", C.c_void_p), ("dz1", C.c_void_p), ("dz2", C.c_void_p), ("w2_dgrad", C.c_void_p), ("w1_dgrad", C.c_void_p),
        ("p1", C.c_void_p), ("p2", C.c_void_p),
        ("sums2", C.c_void_p), ("sums2_replicas", C.c_int32), ("sums2_rstride", C.c_int32),
        ("sums1", C.c_void_p), ("sums1_replicas", C.c_int32), ("sums1_rstride", C.c_int32),
        ("dgamma2", C.c_void_p), ("dbeta2", C.c_void_p)]


DENSE_LAYERS_MAX = 64


class DenseBn1List(C.Structure):
    """saunet_dense_bn1_list"""
    _fields_ = [("count", C.c_int32), ("replicas", C.c_int32), ("sums", C.c_void_p * DENSE_LAYERS_MAX), ("rstride", C.c_int32 * DENSE_LAYERS_MAX),
                ("cin", C.c_int32 * DENSE_LAYERS_MAX), ("dgamma", C.c_void_p * DENSE_LAYERS_MAX), ("dbeta", C.c_void_p * DENSE_LAYERS_MAX)]


class TensorList(C.Structure):
    _fields_ = [("count", C.c_int32), ("ptrs", (C.c_void_p * 96) * 4), ("numel", C.c_int64 * 96)]


class NsItem(C.Structure):
    """saunet_ns_item"""
    _fields_ = [("src", C.c_void_p), ("dst", C.c_void_p), ("buf", C.c_void_p), ("ld_src", C.c_int64), ("ld_dst", C.c_int64),
                ("rows", C.c_int32), ("cols", C.c_int32)]


NS_ITEMS_MAX = 4096


class NsDesc(C.Structure):
    """saunet_ns_desc"""
    _fields_ = [("item", C.c_void_p), ("count", C.c_int32), ("dtype", C.c_int32), ("steps", C.c_int32), ("adjust", C.c_int32),
                ("a", C.c_float), ("b", C.c_float), ("c", C.c_float), ("eps", C.c_float)]


class Int8Desc(C.Structure):
    """saunet_int8_desc"""
    _fields_ = [("a", C.c_void_p), ("a_scale", C.c_void_p), ("lda", C.c_int64), ("m", C.c_int64), ("b", C.c_void_p), ("b_scale", C.c_void_p),
                ("ldb", C.c_int64), ("n", C.c_int32), ("k", C.c_int32), ("bias", C.c_void_p), ("y", C.c_void_p), ("ldy", C.c_int64),
                ("dtype", C.c_int32), ("relu", C.c_int32)]


vp, i32, i64, f32, f64 = C.c_void_p, C.c_int, C.c_int64, C.c_float, C.c_double
_SIGS = {
    "saunet_init": [i32],
    "saunet_pack_weight": [i32, i32, vp, i32, i32, i32, i32, vp, vp],
    "saunet_pack_weight_multi": [C.POINTER(PackList), i32, vp],
    "saunet_conv2d_forward": [C.POINTER(ConvDesc), vp, vp, vp, vp, vp, vp, vp, vp, vp],
    "saunet_conv2d_forward_ex": [C.POINTER(ConvDesc), vp, vp, vp, vp, vp, vp, vp, vp, C.POINTER(BnEpilogue), vp],
    "saunet_conv2d_accumulate_supported": [C.POINTER(ConvDesc)],
    "saunet_conv2d_forward_workspace": [C.POINTER(ConvDesc)],
    "saunet_conv2d_forward_bnpro": [C.POINTER(ConvDesc), vp, vp, vp, C.POINTER(BnPrologue), vp, vp, vp, vp],
    "saunet_bn_xhat": [i32, vp, vp, i32, i32, f64, f32, vp, i32, vp],
    "saunet_conv2d_wgrad": [C.POINTER(ConvDesc), vp, vp, vp, vp, vp, vp, i64, vp],
    "saunet_conv2d_wgrad_bias": [C.POINTER(ConvDesc), vp, vp, vp, vp, vp, vp, vp, i64, vp],
    "saunet_conv2d_wgrad_bias_supported": [C.POINTER(ConvDesc)],
    "saunet_conv2d_wgrad_workspace": [C.POINTER(ConvDesc)],
    "saunet_conv2d_wgrad_deferred": [C.POINTER(ConvDesc), vp, vp, vp, vp, vp, vp, i64, C.POINTER(WgradPending), vp],
    "saunet_wgrad_reduce_multi": [C.POINTER(WgradReduceList), vp],
    "saunet_conv2d_wgrad_grouped_workspace": [C.POINTER(WgradGroup)],
    "saunet_conv2d_wgrad_grouped": [C.POINTER(WgradGroup), vp, i64, vp],
    "saunet_channel_sum": [i32, vp, i64, i32, i32, vp, vp],
    "saunet_bn_stats": [i32, vp, i64, i32, i32, vp, vp, i32, i32, vp],
    "saunet_sum_replicas": [vp, i32, i32, i32, vp],
    "saunet_bn_finalize": [i32, vp, vp, i32, i32, f64, vp, vp, vp, f32, f32, vp, vp, vp, vp, vp, vp, i32, vp],
    "saunet_syncbn_finalize": [i32, vp, vp, i32, i32, f64, vp, vp, f32, f32, vp, vp, vp, vp, vp, vp, vp, vp, vp, vp],
    "saunet_affine_act": [i32, vp, i32, vp, vp, vp, i32, i32, vp, i32, i64, i32, vp],
    "saunet_affine_act_pool": [i32, vp, i32, vp, vp, i32, vp, i32, i64, i32, vp, i32, vp],
    "saunet_bn_backward_reduce": [i32, vp, i32, vp, i32, vp, i32, vp, vp, vp, vp, i32, vp, i32, i32, i64, i32, vp],
    "saunet_bn_backward_apply": [i32, vp, i32, vp, i32, vp, i32, vp, vp, vp, vp, i32, vp, i32, i32, f64, i32, i32,
                                 vp, i32, vp, i32, vp, vp, i64, i32, vp],
    "saunet_affine_act_bn": [i32, vp, i32, C.POINTER(BnPrologue), vp, vp, i32, i32, vp, i32, i64, i32, vp, vp],
    "saunet_affine_act_pool_bn": [i32, vp, i32, C.POINTER(BnPrologue), vp, i32, vp, i32, i64, i32, vp, i32, vp],
    "saunet_bn_relu_avgpool2": [i32, vp, i32, vp, vp, vp, i32, i32, i32, i32, i32, vp],
    "saunet_bn_relu_avgpool2_backward": [i32, vp, i32, vp, i32, vp, vp, vp, vp, i32, vp, i32, vp, i32, i32, i32, i32, i32, i32, vp],
    "saunet_affine_act_mask": [i32, vp, i32, vp, vp, vp, i32, vp, i32, i64, i32, vp, vp],
    "saunet_bn_backward_reduce_masked": [i32, vp, i32, vp, i32, vp, vp, vp, vp, vp, vp, i32, i32, i64, i32, vp],
    "saunet_bn_backward_apply_masked": [i32, vp, i32, vp, i32, vp, vp, vp, vp, vp, vp, i32, i32, f64, i32, i32,
                                        vp, i32, vp, i32, vp, vp, i64, i32, vp],
    "saunet_bn_backward_coeff": [i32, vp, i32, i32, f64, vp, vp, vp, vp, vp, i32, vp],
    "saunet_bn_backward_correct": [i32, vp, i32, vp, i32, vp, vp, vp, vp, i64, i32, vp],
    "saunet_bn_backward_coeff_correct": [i32, i32, vp, i32, i32, f64, vp, vp, vp, vp, vp, vp, vp, vp, i32, vp, i32, i32, i32, vp, vp, i64, vp],
    "saunet_dense_layer_backward_conv2": [C.POINTER(DenseLayerBwd), vp],
    "saunet_dense_layer_backward_conv1": [C.POINTER(DenseLayerBwd), vp],
    "saunet_dense_layer_backward_pair_supported": [C.POINTER(DenseLayerBwd)],
    "saunet_dense_layer_backward_conv1_pair": [C.POINTER(DenseLayerBwd), C.POINTER(DenseLayerBwd), vp],
    "saunet_bn_backward_correct_ab": [i32, vp, i32, vp, i32, vp, i32, vp, i32, i32, i32, f64, vp, vp, i64, i32, vp],
    "saunet_dense_bn1_grads": [C.POINTER(DenseBn1List), vp],
    "saunet_bn_backward_coeff_ab": [i32, vp, i32, i32, vp, vp, i32, vp, vp, vp],
    "saunet_bilinear_forward": [i32, vp, i32, i32, i32, i32, i32, vp, i32, i32, i32, vp],
    "saunet_bilinear_backward": [i32, vp, i32, i32, i32, i32, i32, vp, i32, i32, i32, i32, vp],
    "saunet_im2col": [i32, vp, i32, i32, i32, i32, i32, i32, i32, i32, i32, vp, i32, vp],
    "saunet_pool2x2_forward": [i32, i32, vp, i32, i32, i32, i32, i32, vp, i32, vp],
    "saunet_pool2x2_backward": [i32, i32, vp, vp, i32, i32, i32, i32, i32, i32, vp, i32, i32, vp],
    "saunet_copy_channels": [i32, i32, vp, i32, vp, i32, i64, i32, i32, vp],
    "saunet_sigmoid_forward": [i32, vp, i32, vp, i32, i64, i32, vp],
    "saunet_sigmoid_backward": [i32, vp, i32, vp, i32, vp, i32, i64, i32, i32, vp],
    "saunet_gate_mul_forward": [i32, vp, i32, vp, vp, i32, i64, i32, vp],
    "saunet_gate_mul_backward": [i32, vp, i32, vp, vp, i32, vp, i32, vp, i64, i32, vp],
    "saunet_gate_forward_z": [i32, i32, vp, i32, vp, i32, i64, vp, vp, vp, vp, vp, vp, vp, vp, i32, i32, vp],
    "saunet_gate_forward_out": [i32, i32, vp, i32, vp, i64, vp, vp, vp, i32, vp, vp],
    "saunet_gate_backward_workspace": [i64],
    "saunet_gate_backward_q": [i32, i32, vp, i32, vp, i32, vp, vp, i64, vp, vp, vp, vp, vp, vp, vp, i64, vp],
    "saunet_gate_backward_sums": [i32, i32, vp, i32, vp, i32, vp, vp, i64, vp, vp, vp, vp, vp, vp, vp, vp, vp, vp, vp, vp, i64, vp],
    "saunet_gate_backward_apply": [i32, i32, vp, i32, vp, i32, vp, i32, vp, vp, i64, vp, vp, vp, vp, vp, vp, vp, vp, vp, i32, vp, i32, vp],
    "saunet_expand_coeff": [i32, vp, vp, i32, i32, f64, vp, vp, vp, vp, f32, f32, vp, vp, vp, vp, i32, vp],
    "saunet_expand_forward": [i32, vp, i64, i32, vp, vp, i32, i32, vp],
    "saunet_expand_backward": [i32, vp, i32, vp, i64, i32, vp, vp, i32, vp, i32, i32, vp, vp, vp, vp, vp, vp, vp],
    "saunet_global_avgpool": [i32, vp, i32, i32, i32, i32, vp, vp],
    "saunet_global_pool_workspace": [i32, i32, i32],
    "saunet_global_pool_forward": [i32, i32, vp, i32, i32, i32, i32, vp, vp, vp, i64, vp],
    "saunet_global_pool_backward": [i32, i32, vp, vp, i32, i32, i32, vp, i32, vp],
    "saunet_se_excite": [vp, i32, i32, i32, vp, vp, vp, vp, vp, vp, vp],
    "saunet_se_excite_backward": [vp, vp, vp, vp, i32, i32, i32, vp, vp, vp, vp, vp, vp, vp, vp],
    "saunet_att_combine_forward": [i32, vp, i32, vp, vp, vp, i32, i32, i32, i32, vp],
    "saunet_att_combine_backward": [i32, vp, i32, vp, vp, vp, i32, vp, i32, vp, vp, i32, i32, i32, vp],
    "saunet_add_pooled_grad": [i32, vp, i32, vp, i32, i32, i32, vp],
    "saunet_dual_loss_forward": [i32, vp, i32, vp, vp, vp, i64, vp, vp],
    "saunet_dual_loss_finalize": [vp, i64, vp, vp, vp],
    "saunet_dual_loss_backward": [i32, vp, i32, vp, vp, vp, i64, vp, vp, vp, i32, vp, vp],
    "saunet_softmax_argmax": [i32, vp, i32, i64, i32, vp, i32, vp, vp],
    "saunet_pixel_metrics": [i32, vp, i64, i64, i64, vp, i64, i64, i32, vp, vp, vp],
    "saunet_binary_jaccard": [i32, vp, vp, i64, vp, vp, vp],
    "saunet_canny": [i32, vp, i32, i32, i32, i32, i32, vp, vp, vp],
    "saunet_mask_to_edges": [vp, i32, i32, i32, i32, vp, vp],
    "saunet_labels_uncrop_resize": [vp] + [i32] * 13 + [vp, vp],
    "saunet_augment_geometric": [vp, vp, i32, i32, i32, vp, i32, vp, vp, vp],
    "saunet_augment_gamma_zscore": [vp, i32, i32, vp, vp],
    "saunet_uniform_noise": [C.c_uint64, vp, i64, vp],
    "saunet_gauss_blur": [vp, vp, vp, i32, i32, i32, vp, i32, i32, f32, vp],
    "saunet_elastic_warp": [vp, vp, vp, vp, vp, i32, i32, i32, vp, vp, vp, vp, vp],
    "saunet_sgd_step": [C.POINTER(TensorList), vp, vp],
    "saunet_radam_step": [C.POINTER(TensorList), vp, vp],
    "saunet_adam_step": [C.POINTER(TensorList), vp, vp],
    "saunet_newton_schulz_workspace": [C.POINTER(NsDesc)],
    "saunet_newton_schulz": [C.POINTER(NsDesc), vp, i64, vp],
    "saunet_muon_step": [C.POINTER(NsDesc), vp, vp, i64, vp],
    "saunet_quantize_rows": [i32, vp, i64, i64, i32, vp, vp, i32, vp, i64, vp, vp],
    "saunet_matmul_int8": [C.POINTER(Int8Desc), vp],
    "saunet_linear_int8": [C.POINTER(Int8Desc), i32, vp, i64, vp, i64, vp],
    "saunet_bucket_copy": [C.POINTER(TensorList), i32, f32, vp],
}
ABI_VERSION = 4          # include/saunet_hip.h: SAUNET_ABI_VERSION (the struct layouts below mirror that header)
EXPORTS = sorted(list(_SIGS) + ["saunet_last_error", "saunet_version", "saunet_launch_log"])

_lib = None


def load():
    """Load the shared library (never falls back to anything else)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError("libsaunet_hip.so is not built (%s). Run __graft_entry__.build() / "
                           "python -m saunet_amd._build; there is no CPU or PyTorch fallback." % LIB_PATH)
    lib = C.CDLL(LIB_PATH)
    lib.saunet_last_error.restype = C.c_char_p
    lib.saunet_version.restype = C.c_int
    lib.saunet_launch_log.restype = C.c_char_p
    if lib.saunet_version() != ABI_VERSION:
        raise RuntimeError("%s speaks ABI version %d, this binding (include/saunet_hip.h: SAUNET_ABI_VERSION) %d: rebuild the library"
                           % (LIB_PATH, lib.saunet_version(), ABI_VERSION))
    for name, sig in _SIGS.items():
        fn = getattr(lib, name)
        fn.argtypes = sig
        fn.restype = C.c_int64 if name.endswith("_workspace") else C.c_int
    _lib = lib
    return lib


def _check(rc, name):
    if rc != 0:
        raise RuntimeError("%s failed (%d): %s" % (name, rc, _lib.saunet_last_error().decode()))


def call(name, *args):
    lib = load()
    rc = getattr(lib, name)(*args)
    if rc != 0:
        _check(rc, name)


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_cur_device = getattr(torch._C, "_cuda_getDevice", None)


def stream():
    """raw handle of the current HIP stream of the current device (the C ABI takes it as void*).  The two private torch._C getters are what
    torch.cuda.current_stream() wraps; called directly they cost 0.3 us instead of 9 us -- 1 200 launches per eager step (3.7 ms of host time)."""
    if _raw_stream is not None and _cur_device is not None:
        return _raw_stream(_cur_device())
    return torch.cuda.current_stream().cuda_stream


class _Here:
    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


_HERE_CTX = _Here()


def on(device):
    """context that makes `device` the current one -- nothing to do, at no cost, where it already is"""
    if _cur_device is not None and _cur_device() == device.index:
        return _HERE_CTX
    return torch.cuda.device(device)


def ptr(t):
    return None if t is None else t.data_ptr()


def matrix_dtype_code(t):
    """storage type of the matrix operators (newton_schulz, the int8 products): float16 too"""
    return F16 if t.dtype == torch.float16 else dtype_code(t)


def dtype_code(t):
    if t.dtype == torch.float32:
        return F32
    if t.dtype == torch.bfloat16:
        return BF16
    raise RuntimeError("saunet_amd: unsupported activation dtype %s" % t.dtype)
