"""ctypes binding of libv1t_amd.so (the C-ABI in include/v1t_amd.h).

The product path has NO CPU / eager fallback: if the HIP library is missing or a launch fails,
the ops raise RuntimeError (the reference's OOM probe, utils/utils.py:460, relies on RuntimeError).
PyTorch is used only for device memory and streams: tensors are passed as raw device pointers.
"""
from __future__ import annotations

import ctypes as C
import os
import typing as t

import torch
from torch.autograd import forward_ad

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "lib", os.environ.get("V1T_LIB", "libv1t_amd.so"))  # V1T_LIB (dev): an experiment build next to it

c_void_p, c_int, c_ll, c_float, c_u64, c_u32 = C.c_void_p, C.c_int, C.c_longlong, C.c_float, C.c_uint64, C.c_uint32


class VitConfig(C.Structure):
    _fields_ = [
        ("in_channels", c_int), ("in_h", c_int), ("in_w", c_int),
        ("patch_size", c_int), ("patch_stride", c_int), ("patch_mode", c_int),
        ("emb_dim", c_int), ("num_heads", c_int), ("mlp_dim", c_int), ("num_blocks", c_int),
        ("behavior_mode", c_int), ("num_mice", c_int), ("use_lsa", c_int), ("use_bias", c_int),
        ("p_dropout", c_float), ("t_dropout", c_float), ("ln_eps", c_float),
        ("core_kind", c_int), ("conv_pad", c_int), ("pos_mode", c_int),
    ]


class TailUnit(C.Structure):
    """`v1t_tail_unit` (include/v1t_amd.h): one local mouse-batch of a training step's readout tail."""
    _fields_ = [
        ("n_images", c_int), ("n_neurons", c_int), ("image_offset", c_int), ("grid_dim", c_int),
        ("eps_stream", c_u32), ("fill_eps", c_int), ("loss_scale", c_float), ("feat_stride", c_int),
        ("pupil", c_void_p), ("response", c_void_p),
        ("sp", c_void_p * 6), ("dsp", c_void_p * 6),
        ("src", c_void_p), ("gp", c_void_p * 4), ("dgp", c_void_p * 4),
        ("mu", c_void_p), ("dmu", c_void_p), ("sigma", c_void_p), ("dsigma", c_void_p),
        ("feat", c_void_p), ("dfeat", c_void_p), ("bias", c_void_p), ("dbias", c_void_p),
        ("shift", c_void_p), ("dshift", c_void_p),
        ("eps", c_void_p), ("grid", c_void_p), ("dgrid", c_void_p),
        ("u", c_void_p), ("yhat", c_void_p), ("du", c_void_p), ("loss", c_void_p),
        ("rws", c_void_p), ("rws_bytes", c_ll), ("gws", c_void_p), ("gws_bytes", c_ll),
    ]


class AdamRange(C.Structure):
    """`v1t_adam_range`: one (arena range, learning rate, L1 coefficient) piece of `v1t_adamw_multi`."""
    _fields_ = [("p", c_void_p), ("g", c_void_p), ("m", c_void_p), ("v", c_void_p), ("n", c_ll), ("lr", c_float), ("l1", c_float), ("step", c_int), ("pad_", c_int)]


class RotaryOperand(C.Structure):
    """`v1t_rotary_operand`: one tensor of `v1t_rotary`, its strides in elements."""
    _fields_ = [("x", c_void_p), ("y", c_void_p), ("xb", c_ll), ("xt", c_ll), ("xh", c_ll), ("yb", c_ll), ("yt", c_ll), ("yh", c_ll), ("heads", c_int), ("y_room", c_int)]


class Matrix(C.Structure):
    """`v1t_matrix`: one update of `v1t_orthogonalize`."""
    _fields_ = [("in_", c_void_p), ("out", c_void_p), ("row_stride", c_ll), ("col_stride", c_ll), ("rows", c_int), ("cols", c_int)]


class MuonRange(C.Structure):
    """`v1t_muon_range`: one matrix of `v1t_muon_step`."""
    _fields_ = [("p", c_void_p), ("g", c_void_p), ("m", c_void_p), ("rows", c_int), ("cols", c_int), ("lr", c_float), ("decay", c_float), ("l1", c_float), ("pad_", c_int)]


# name -> (restype, argtypes); every symbol declared in include/v1t_amd.h
SIGNATURES: t.Dict[str, t.Tuple[t.Any, t.List[t.Any]]] = {
    "v1t_abi_version": (c_int, []),
    "v1t_tails_prepare": (c_int, [C.POINTER(TailUnit), c_int, c_u64, c_int, c_int, c_void_p]),
    "v1t_tails_forward": (c_int, [C.POINTER(TailUnit), c_int, c_void_p, c_void_p, c_ll, c_ll, c_int, c_int, c_int, c_void_p, c_void_p]),
    "v1t_tails_backward": (c_int, [C.POINTER(TailUnit), c_int, c_void_p, c_ll, c_ll, c_int, c_int, c_int, c_void_p]),
    "v1t_adamw_multi": (c_int, [C.POINTER(AdamRange), c_int, c_float, c_float, c_float, c_float, c_int, c_void_p]),
    "v1t_fill_zero": (c_int, [c_void_p, c_ll, c_void_p]),
    "v1t_inputs_multi": (c_int, [C.POINTER(c_void_p), C.POINTER(c_void_p), C.POINTER(c_void_p), C.POINTER(c_int), c_int, c_int, c_int, c_int, c_void_p, c_int, c_int,
                                 c_void_p, c_int, c_int, c_void_p]),
    "v1t_mfma_peak_probe": (c_int, [c_int, c_int, C.POINTER(C.c_double), C.POINTER(C.c_double), C.POINTER(C.c_double), c_void_p]),
    "v1t_error_string": (C.c_char_p, [c_int]),
    "v1t_vit_create": (c_int, [C.POINTER(VitConfig), C.POINTER(c_void_p)]),
    "v1t_vit_destroy": (None, [c_void_p]),
    "v1t_vit_set_rotary": (c_int, [c_void_p, c_void_p, C.POINTER(c_int), c_int, C.c_double]),
    "v1t_vit_arena_floats": (c_ll, [c_void_p]),
    "v1t_vit_param_floats": (c_ll, [c_void_p]),
    "v1t_vit_num_tensors": (c_int, [c_void_p]),
    "v1t_vit_tensor_info": (c_int, [c_void_p, c_int, C.c_char_p, c_int, C.POINTER(c_ll), C.POINTER(c_int), C.POINTER(c_ll), C.POINTER(c_int)]),
    "v1t_vit_tokens": (c_int, [c_void_p]),
    "v1t_vit_cls_tokens": (c_int, [c_void_p]),
    "v1t_vit_padded_dim": (c_int, [c_void_p]),
    "v1t_vit_grid_h": (c_int, [c_void_p]),
    "v1t_vit_grid_w": (c_int, [c_void_p]),
    "v1t_vit_shadow_bytes": (c_ll, [c_void_p]),
    "v1t_vit_workspace_bytes": (c_ll, [c_void_p, c_int, c_int]),
    "v1t_vit_scratch_bytes": (c_ll, [c_void_p, c_int]),
    "v1t_vit_workspace_offset": (c_ll, [c_void_p, c_int, c_int, C.c_char_p, c_int]),
    "v1t_vit_pack": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p]),
    "v1t_vit_forward": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_void_p, c_ll, c_int, c_int, c_u64, c_void_p, c_void_p, c_void_p]),
    "v1t_vit_backward": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_void_p, c_void_p, c_ll, c_int, c_u64, c_void_p, c_void_p, c_void_p, c_void_p]),
    "v1t_vit_backward_events": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_void_p, c_void_p, c_ll, c_int, c_u64, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p]),
    "v1t_dropout_mask": (c_int, [c_u64, c_u32, c_float, c_ll, c_ll, c_void_p, c_void_p]),
    "v1t_attention_dropout_rate": (c_float, [c_float]),
    "v1t_vit_scratch_bytes_input": (c_ll, [c_void_p, c_int]),
    "v1t_vit_backward_input": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_void_p, c_void_p, c_ll, c_int, c_u64, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p]),
    "v1t_vit_backward_second_stream": (c_int, [c_void_p, c_int]),
    "v1t_gaussian2d_forward": (c_int, [c_void_p, c_ll, c_ll, c_int, c_int, c_int, c_int, c_int, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p]),
    "v1t_gaussian2d_backward": (c_int, [c_void_p, c_ll, c_ll, c_int, c_int, c_int, c_int, c_int, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_ll, c_ll, c_void_p, c_void_p, c_void_p, c_void_p]),
    "v1t_gather_transform": (c_int, [c_void_p, c_int, c_void_p, c_int, c_ll, c_void_p, c_ll, c_void_p, c_ll, c_void_p, c_ll, c_int, c_void_p, c_void_p]),
    "v1t_metrics_accumulate": (c_int, [c_void_p, c_void_p, c_int, c_int, c_float, c_void_p, c_void_p, c_void_p]),
    "v1t_metrics_correlation": (c_int, [c_void_p, c_ll, c_int, c_float, c_void_p, c_void_p, c_void_p]),
    "v1t_metrics_group_accumulate": (c_int, [c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p, c_void_p, c_void_p]),
    "v1t_metrics_group_finalize": (c_int, [c_void_p, c_void_p, c_void_p, c_int, c_int, c_float, c_void_p, c_void_p, c_void_p, c_void_p]),
    "v1t_crop_nearest": (c_int, [c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_void_p, c_void_p, c_int, c_int, c_void_p]),
    "v1t_resize_bilinear": (c_int, [c_void_p, c_int, c_int, c_int, c_void_p, c_int, c_int, c_void_p]),
    "v1t_resize_bilinear_backward": (c_int, [c_void_p, c_int, c_int, c_int, c_void_p, c_int, c_int, c_void_p]),
    "v1t_gaussian2d_backward_ws_bytes": (c_ll, [c_int, c_int, c_int, c_int]),
    "v1t_gaussian2d_backward_ws": (c_int, [c_void_p, c_ll, c_ll, c_int, c_int, c_int, c_int, c_int, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_ll, c_ll, c_void_p, c_void_p, c_void_p, c_void_p, c_ll, c_void_p]),
    "v1t_gaussian2d_backward_parts": (c_int, [c_void_p, c_ll, c_ll, c_int, c_int, c_int, c_int, c_int, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_ll, c_ll, c_void_p, c_void_p, c_void_p, c_void_p, c_ll, c_int, c_void_p]),
    "v1t_readout_grid_forward": (c_int, [c_int, c_int, c_int] + [c_void_p] * 11),
    "v1t_readout_grid_backward": (c_int, [c_int, c_int, c_int] + [c_void_p] * 17),
    "v1t_normal_fill": (c_int, [c_void_p, c_ll, c_u64, c_u32, c_void_p]),
    "v1t_concat2": (c_int, [c_void_p, c_int, c_void_p, c_int, c_int, c_void_p, c_int, c_void_p]),
    "v1t_core_shifter_forward": (c_int, [c_int] + [c_void_p] * 9),
    "v1t_core_shifter_backward": (c_int, [c_int] + [c_void_p] * 15),
    "v1t_elu1_poisson": (c_int, [c_void_p, c_void_p, c_ll, c_float, c_float, c_void_p, c_void_p, c_void_p, c_void_p]),
    "v1t_poisson_loss": (c_int, [c_void_p, c_void_p, c_ll, c_float, c_float, c_void_p, c_void_p, c_void_p]),
    "v1t_elu1_backward": (c_int, [c_void_p, c_void_p, c_void_p, c_ll, c_void_p, c_void_p]),
    "v1t_readout_grid_backward_ws_bytes": (c_ll, [c_int, c_int]),
    "v1t_readout_grid_backward_ws": (c_int, [c_int, c_int, c_int] + [c_void_p] * 16 + [c_void_p, c_ll, c_void_p]),
    "v1t_adamw_step": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_ll, c_float, c_float, c_float, c_float, c_float, c_int, c_float, c_int, c_void_p]),
    "v1t_l1_sum": (c_int, [c_void_p, c_ll, c_float, c_void_p, c_void_p]),
    "v1t_l1_grad": (c_int, [c_void_p, c_void_p, c_ll, c_float, c_void_p]),
    "v1t_l1_grad_dev": (c_int, [c_void_p, c_void_p, c_ll, c_float, c_void_p, c_void_p]),
    "v1t_gemm_nt": (c_int, [c_void_p, c_int, c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_int, c_int, c_void_p]),
    "v1t_gemm_tn": (c_int, [c_void_p, c_int, c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_int, c_int, c_void_p]),
    "v1t_gemm_tn_slab_bytes": (c_ll, [c_int, c_int, c_int, c_int]),
    "v1t_gemm_tn_slab": (c_int, [c_void_p, c_int, c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_int, c_int, c_void_p, c_ll, c_void_p]),
    "v1t_attention_forward": (c_int, [c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_int, c_int, c_float, c_u64, c_u32, c_void_p, c_void_p, c_void_p]),
    "v1t_attention_backward": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_int, c_int, c_float, c_u64, c_u32, c_void_p, c_void_p, c_void_p, c_void_p]),
    "v1t_attention_backward_ws_bytes": (c_ll, [c_int, c_int, c_int]),
    "v1t_attention_forward_f16o": (c_int, [c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_int, c_int, c_float, c_u64, c_u32, c_void_p, c_void_p, c_void_p]),
    "v1t_attention_backward_ws_f16o": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_int, c_int, c_float, c_u64, c_u32, c_void_p, c_void_p, c_void_p, c_void_p, c_ll, c_void_p]),
    "v1t_attention_backward_ws": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_int, c_int, c_float, c_u64, c_u32, c_void_p, c_void_p, c_void_p, c_void_p, c_ll, c_void_p]),
    "v1t_rollout_headmax": (c_int, [c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_int, c_int, c_void_p, c_int, c_void_p, c_void_p]),
    "v1t_rollout_headmax_rows": (c_int, [c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_int, c_int, c_void_p, c_int, c_void_p, c_int, c_void_p]),
    "v1t_attention_probs": (c_int, [c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_int, c_int, c_void_p, c_int, c_void_p]),
    "v1t_rollout_vecmat": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p]),
    "v1t_rollout_matmul": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p]),
    "v1t_rotary": (c_int, [C.POINTER(RotaryOperand), c_int, c_int, c_int, c_int, c_int, C.POINTER(c_int), c_int, C.c_double, c_int, c_int, c_int, c_void_p, c_int,
                           c_ll, c_ll, c_ll, c_void_p]),
    "v1t_orthogonalize_ws_bytes": (c_ll, [C.POINTER(c_int), C.POINTER(c_int), c_int]),
    "v1t_orthogonalize": (c_int, [C.POINTER(Matrix), c_int, c_int, c_int, C.POINTER(c_float), c_float, c_void_p, c_ll, c_void_p]),
    "v1t_muon_step": (c_int, [C.POINTER(MuonRange), c_int, c_float, c_int, c_int, C.POINTER(c_float), c_float, c_int, c_void_p, c_ll, c_void_p]),
    "v1t_profile_enable": (c_int, [c_int, c_int]),
    "v1t_profile_read": (c_int, [C.POINTER(c_int), C.POINTER(C.c_double)]),
    "v1t_layernorm_forward": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_float, c_void_p]),
    "v1t_layernorm_backward": (c_int, [c_void_p] * 12 + [c_int, c_int, c_int, c_int, c_void_p]),
}

_lib: t.Optional[C.CDLL] = None


def load() -> C.CDLL:
    """dlopen the in-tree library; raises RuntimeError (never falls back) when it is missing."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(
            f"v1t_amd: HIP library {LIB_PATH} not found — build it with `python -m v1t_amd.build` "
            "(hipcc --offload-arch=gfx950). There is no CPU fallback."
        )
    # the product library and the experiment build are content-checked; any other V1T_LIB (a one-off A/B build) is loaded as it is
    checked = os.environ.get("V1T_LIB") in (None, "libv1t_amd.so", "libv1t_amd_exp.so")
    if checked and not os.environ.get("V1T_ALLOW_STALE_LIB"):
        # the git-ignored .so travels with the repo snapshot: refuse one that was built from other sources than the tree holds (content
        # hash over every .hip / .h and the flags, v1t_amd/build.py) instead of silently testing / timing old kernels
        from . import build as _b

        if not _b.is_current(LIB_PATH):
            raise RuntimeError(f"v1t_amd: {LIB_PATH} was built from other sources than the tree holds (built {_b.buildinfo(LIB_PATH).get('sources_sha16')}, "
                               f"tree {_b.sources_sha16()}): run `python -m v1t_amd.build`. There is no CPU fallback.")
    lib = C.CDLL(LIB_PATH)
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)  # AttributeError if the .so does not export a declared symbol
        fn.restype = res
        fn.argtypes = args
    _lib = lib
    return lib


def check(code: int, what: str = "") -> None:
    if code != 0:
        msg = load().v1t_error_string(code).decode()
        raise RuntimeError(f"v1t_amd {what}: {msg} (code {code})")


def ptr(x: t.Optional[torch.Tensor]) -> t.Optional[int]:
    return None if x is None else x.data_ptr()


def stream() -> int:
    return torch.cuda.current_stream().cuda_stream


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # current_stream().cuda_stream without the Python object: 0.3 instead of 3 us


def stream_of(device: int) -> int:
    return _raw_stream(device) if _raw_stream is not None else torch.cuda.current_stream(device).cuda_stream


def require_cuda(x: torch.Tensor, what: str) -> None:
    if not x.is_cuda:
        raise RuntimeError(f"v1t_amd {what}: tensor is on {x.device}; the HIP path needs a GPU tensor (no CPU fallback).")


def dual_level() -> bool:
    """Whether tensors may carry a tangent (torch.autograd.forward_ad)."""
    return getattr(forward_ad, "_current_level", 0) >= 0


def refuse_tangents(what: str, tensors) -> None:
    """Called within a dual level by operators whose kernels read and write raw pointers: a dual tensor's tangent would be lost without a word, which reads as a
    derivative of zero."""
    if any(x is not None and forward_ad.unpack_dual(x).tangent is not None for x in tensors):
        raise NotImplementedError(f"v1t_amd {what}: forward-mode differentiation is not supported (a tensor carries a tangent)")


def leaves_in_capture(out: torch.Tensor, what: str) -> None:
    """Called by an operator with its differentiable result. The node that receives a leaf's gradient belongs to
    the stream of the first pass that used the leaf, for as long as any graph of that pass lives; a backward pass captured meanwhile on another
    stream would wait on that stream inside the capture, which ends the process when the capture ends. So an eager pass marks the node with its
    stream, and a captured pass that finds another stream's mark is refused."""
    here = stream_of(out.get_device())
    for node, _ in out.grad_fn.next_functions:
        if hasattr(node, "variable") and node.metadata.setdefault("v1t_stream", here) != here and torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"v1t_amd {what}: a graph of an earlier pass over the same leaf tensor is still alive on another stream; its backward cannot be "
                               "captured beside it. Drop that pass's outputs (del) before the capture.")


def grad_sink(p):
    """Where a backward kernel that ACCUMULATES (+=) should write the gradient of leaf tensor `p`, and what the
    autograd Function should return for it: straight into ``p.grad`` when that exists as a dense fp32 tensor (the
    flat-arena views the trainer attaches: no zero-fill, no AccumulateGrad add kernel), else a fresh zeroed buffer."""
    import torch

    g = getattr(p, "grad", None)
    if p.is_leaf and g is not None and g.dtype == torch.float32 and g.shape == p.shape and g.is_contiguous() and g.device == p.device:
        return g, None
    z = torch.zeros_like(p)
    return z, z
