"""ctypes mirror of the C ABI in include/convnd_hip.h.

The PyTorch operators call the C ABI from C++ (csrc/torch_ops.cpp); this module exposes
the same entry points to Python for diagnostics, tests and callers that manage device
memory themselves (pointers and a hipStream_t as integers).
"""

import ctypes

MAX_RANK = 62

FLOAT32, FLOAT64, FLOAT16, BFLOAT16 = 0, 1, 2, 3
SUCCESS, INVALID_ARGUMENT, WORKSPACE_TOO_SMALL, LAUNCH_FAILED, UNSUPPORTED = 0, 1, 2, 3, 4

# Every extern "C" symbol the header declares.
EXPORTED_SYMBOLS = (
    "convnd_hip_last_error",
    "convnd_hip_validate",
    "convnd_hip_forward_workspace_size",
    "convnd_hip_forward",
    "convnd_hip_backward_workspace_size",
    "convnd_hip_backward",
    "convnd_hip_plan_name",
    "convnd_hip_plan_describe",
    "convnd_hip_timing_enable",
    "convnd_hip_timing_read",
    "convnd_hip_partial_rescale",
    "convnd_hip_partial_count",
    "convnd_hip_forward_act",
    "convnd_hip_forward_noalloc",
    "convnd_hip_plan_check",
    "convnd_hip_forward_workspace_size_layout",
    "convnd_hip_backward_workspace_size_layout",
    "convnd_hip_forward_layout",
    "convnd_hip_backward_layout",
    "convnd_hip_layer_norm",
    "convnd_hip_layer_norm_backward_workspace_size",
    "convnd_hip_layer_norm_backward",
    "convnd_hip_linear_workspace_size",
    "convnd_hip_linear",
    "convnd_hip_linear_backward_workspace_size",
    "convnd_hip_linear_backward",
    "convnd_hip_linear_plan_describe",
    "convnd_hip_recurrence_carries",
    "convnd_hip_recurrence_workspace_size",
    "convnd_hip_recurrence",
    "convnd_hip_recurrence_backward",
    "convnd_hip_recurrence_plan_describe",
    "convnd_hip_gated_linear_workspace_size",
    "convnd_hip_gated_linear_kept_size",
    "convnd_hip_gated_linear",
    "convnd_hip_gated_linear_backward_workspace_size",
    "convnd_hip_gated_linear_backward",
    "convnd_hip_delta_saved",
    "convnd_hip_delta_workspace_size",
    "convnd_hip_delta",
    "convnd_hip_delta_backward_workspace_size",
    "convnd_hip_delta_backward",
    "convnd_hip_delta_plan_describe",
)

CHANNELS_FIRST, CHANNELS_LAST, CHANNELS_LAST_INPUT = 0, 1, 2

# Bytes of the per-GPU static scratch of convnd_hip_forward_noalloc (CONVND_HIP_NOALLOC_SCRATCH_BYTES).
NOALLOC_SCRATCH_BYTES = 64 << 20


class Problem(ctypes.Structure):
    """struct convnd_hip_problem."""

    _fields_ = [
        ("rank", ctypes.c_int64),
        ("batch", ctypes.c_int64),
        ("channels", ctypes.c_int64),
        ("output_channels", ctypes.c_int64),
        ("groups", ctypes.c_int64),
        ("input", ctypes.c_int64 * MAX_RANK),
        ("kernel", ctypes.c_int64 * MAX_RANK),
        ("stride", ctypes.c_int64 * MAX_RANK),
        ("padding", ctypes.c_int64 * MAX_RANK),
        ("dilation", ctypes.c_int64 * MAX_RANK),
    ]

    @classmethod
    def make(cls, x_shape, w_shape, stride, padding, dilation, groups=1):
        rank = len(x_shape) - 2
        p = cls()
        p.rank, p.batch, p.channels, p.output_channels, p.groups = (
            rank, x_shape[0], x_shape[1], w_shape[0], groups,
        )
        for a in range(rank):
            p.input[a], p.kernel[a] = x_shape[a + 2], w_shape[a + 2]
            p.stride[a], p.padding[a], p.dilation[a] = stride[a], padding[a], dilation[a]
        return p


class LinearProblem(ctypes.Structure):
    """struct convnd_hip_linear_problem."""

    _fields_ = [
        (name, ctypes.c_int64)
        for name in ("rows", "inputs", "outputs", "input_stride", "residual_stride", "grad_stride")
    ] + [("activation", ctypes.c_int)]


class RecurrenceProblem(ctypes.Structure):
    """struct convnd_hip_recurrence_problem."""

    _fields_ = [
        (name, ctypes.c_int64)
        for name in ("batch", "tokens", "channels", "input_batch", "input_token", "gate_batch", "gate_token")
    ] + [("wide_lengths", ctypes.c_int)]


class DeltaProblem(ctypes.Structure):
    """struct convnd_hip_delta_problem."""

    _fields_ = [
        (name, ctypes.c_int64) for name in ("batch", "tokens", "key_heads", "heads", "key_size", "value_size")
    ] + [
        (f"{tensor}_{axis}", ctypes.c_int64)
        for tensor in ("query", "key", "value", "decay", "beta", "grad")
        for axis in ("batch", "token", "head")
    ] + [
        ("scale", ctypes.c_double),
        ("normalize", ctypes.c_int),
        ("gate_dtype", ctypes.c_int),
        ("wide_lengths", ctypes.c_int),
    ]

    @classmethod
    def make(cls, batch, tokens, key_heads, heads, key_size, value_size, gate_dtype):
        """Of contiguous tensors; scale 1."""
        p = cls(batch=batch, tokens=tokens, key_heads=key_heads, heads=heads, key_size=key_size,
                value_size=value_size, gate_dtype=gate_dtype, scale=1.0)
        for name, count, size in (("query", key_heads, key_size), ("key", key_heads, key_size),
                                  ("value", heads, value_size), ("grad", heads, value_size),
                                  ("decay", heads, 1), ("beta", heads, 1)):
            setattr(p, f"{name}_batch", tokens * count * size)
            setattr(p, f"{name}_token", count * size)
            setattr(p, f"{name}_head", size)
        return p


def bind(library: ctypes.CDLL) -> ctypes.CDLL:
    """Declare argument and result types on a loaded libconvnd_hip.so."""
    P = ctypes.POINTER(Problem)
    vp, sz, i64 = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int64
    library.convnd_hip_last_error.restype = ctypes.c_char_p
    library.convnd_hip_last_error.argtypes = []
    library.convnd_hip_validate.restype = ctypes.c_int
    library.convnd_hip_validate.argtypes = [P, i64, i64, ctypes.POINTER(i64)]
    library.convnd_hip_forward_workspace_size.restype = sz
    library.convnd_hip_forward_workspace_size.argtypes = [P, ctypes.c_int]
    library.convnd_hip_forward.restype = ctypes.c_int
    library.convnd_hip_forward.argtypes = [P, ctypes.c_int, vp, vp, vp, vp, vp, sz, vp]
    library.convnd_hip_backward_workspace_size.restype = sz
    library.convnd_hip_backward_workspace_size.argtypes = [P, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int]
    library.convnd_hip_backward.restype = ctypes.c_int
    library.convnd_hip_backward.argtypes = [P, ctypes.c_int, vp, vp, vp, vp, vp, vp, vp, sz, vp]
    library.convnd_hip_plan_name.restype = ctypes.c_char_p
    library.convnd_hip_plan_name.argtypes = [P, ctypes.c_int, ctypes.c_int]
    library.convnd_hip_plan_describe.restype = ctypes.c_int
    library.convnd_hip_plan_describe.argtypes = [P, ctypes.c_int, ctypes.c_int, ctypes.c_char_p, sz]
    library.convnd_hip_timing_enable.restype = ctypes.c_int
    library.convnd_hip_timing_enable.argtypes = [ctypes.c_int]
    library.convnd_hip_timing_read.restype = ctypes.c_int
    library.convnd_hip_timing_read.argtypes = [ctypes.c_int, ctypes.POINTER(ctypes.c_double), ctypes.POINTER(i64)]
    library.convnd_hip_forward_act.restype = ctypes.c_int
    library.convnd_hip_forward_act.argtypes = [P, ctypes.c_int, vp, vp, vp, vp, ctypes.c_int, vp, sz, vp]
    library.convnd_hip_plan_check.restype = ctypes.c_int
    library.convnd_hip_plan_check.argtypes = [P, ctypes.c_int]
    library.convnd_hip_forward_noalloc.restype = ctypes.c_int
    library.convnd_hip_forward_noalloc.argtypes = [P, ctypes.c_int, vp, vp, vp, vp, vp]
    library.convnd_hip_forward_workspace_size_layout.restype = sz
    library.convnd_hip_forward_workspace_size_layout.argtypes = [P, ctypes.c_int, ctypes.c_int]
    library.convnd_hip_backward_workspace_size_layout.restype = sz
    library.convnd_hip_backward_workspace_size_layout.argtypes = [
        P, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int
    ]
    library.convnd_hip_forward_layout.restype = ctypes.c_int
    library.convnd_hip_forward_layout.argtypes = [P, ctypes.c_int, ctypes.c_int, ctypes.c_int, vp, vp, vp, vp, vp, sz, vp]
    library.convnd_hip_backward_layout.restype = ctypes.c_int
    library.convnd_hip_backward_layout.argtypes = [P, ctypes.c_int, ctypes.c_int, vp, vp, vp, vp, vp, vp, vp, sz, vp]
    library.convnd_hip_partial_count.restype = ctypes.c_int
    library.convnd_hip_partial_count.argtypes = [P, ctypes.c_int, vp, vp, vp]
    library.convnd_hip_partial_rescale.restype = ctypes.c_int
    library.convnd_hip_partial_rescale.argtypes = [
        ctypes.c_int, vp, vp, vp, vp, i64, i64, i64, i64, i64, ctypes.c_double, vp
    ]
    R, dbl = ctypes.POINTER(RecurrenceProblem), ctypes.c_double
    library.convnd_hip_layer_norm.restype = ctypes.c_int
    library.convnd_hip_layer_norm.argtypes = [
        ctypes.c_int, ctypes.c_int, vp, i64, vp, vp, vp, vp, vp, i64, i64, dbl, vp
    ]
    library.convnd_hip_layer_norm_backward_workspace_size.restype = sz
    library.convnd_hip_layer_norm_backward_workspace_size.argtypes = [ctypes.c_int, i64, i64]
    library.convnd_hip_layer_norm_backward.restype = ctypes.c_int
    library.convnd_hip_layer_norm_backward.argtypes = [
        ctypes.c_int, ctypes.c_int, vp, i64, vp, i64, vp, vp, vp, vp, vp, vp, i64, i64, vp, sz, vp
    ]
    L = ctypes.POINTER(LinearProblem)
    library.convnd_hip_linear_workspace_size.restype = sz
    library.convnd_hip_linear_workspace_size.argtypes = [ctypes.c_int, L, vp, vp]
    library.convnd_hip_linear.restype = ctypes.c_int
    library.convnd_hip_linear.argtypes = [ctypes.c_int, L, vp, vp, vp, vp, vp, vp, vp, sz, vp]
    library.convnd_hip_linear_backward_workspace_size.restype = sz
    library.convnd_hip_linear_backward_workspace_size.argtypes = [
        ctypes.c_int, L, vp, vp, vp, ctypes.c_int, ctypes.c_int, ctypes.c_int
    ]
    library.convnd_hip_linear_backward.restype = ctypes.c_int
    library.convnd_hip_linear_backward.argtypes = [
        ctypes.c_int, L, vp, vp, vp, vp, vp, vp, vp, vp, sz, vp
    ]
    library.convnd_hip_gated_linear_workspace_size.restype = sz
    library.convnd_hip_gated_linear_workspace_size.argtypes = [ctypes.c_int, L, vp, vp]
    library.convnd_hip_gated_linear_kept_size.restype = sz
    library.convnd_hip_gated_linear_kept_size.argtypes = [ctypes.c_int, L]
    library.convnd_hip_gated_linear.restype = ctypes.c_int
    library.convnd_hip_gated_linear.argtypes = [ctypes.c_int, L, vp, vp, vp, vp, vp, vp, sz, vp]
    library.convnd_hip_gated_linear_backward_workspace_size.restype = sz
    library.convnd_hip_gated_linear_backward_workspace_size.argtypes = [
        ctypes.c_int, L, vp, vp, ctypes.c_int, ctypes.c_int, ctypes.c_int
    ]
    library.convnd_hip_gated_linear_backward.restype = ctypes.c_int
    library.convnd_hip_gated_linear_backward.argtypes = [
        ctypes.c_int, L, vp, vp, vp, vp, vp, vp, vp, vp, sz, vp
    ]
    library.convnd_hip_recurrence_carries.restype = i64
    library.convnd_hip_recurrence_carries.argtypes = [i64]
    library.convnd_hip_recurrence_workspace_size.restype = sz
    library.convnd_hip_recurrence_workspace_size.argtypes = [ctypes.c_int, R]
    library.convnd_hip_recurrence.restype = ctypes.c_int
    library.convnd_hip_recurrence.argtypes = [ctypes.c_int, R, vp, vp, vp, vp, vp, vp, vp, vp, sz, vp]
    library.convnd_hip_recurrence_backward.restype = ctypes.c_int
    library.convnd_hip_recurrence_backward.argtypes = [
        ctypes.c_int, R, vp, vp, vp, vp, vp, vp, vp, vp, vp, vp, sz, vp
    ]
    D = ctypes.POINTER(DeltaProblem)
    library.convnd_hip_delta_saved.restype = i64
    library.convnd_hip_delta_saved.argtypes = [ctypes.c_int, D]
    library.convnd_hip_delta_workspace_size.restype = sz
    library.convnd_hip_delta_workspace_size.argtypes = [ctypes.c_int, D, vp, vp, vp, ctypes.c_int]
    library.convnd_hip_delta.restype = ctypes.c_int
    library.convnd_hip_delta.argtypes = [ctypes.c_int, D, *[vp] * 11, sz, vp]
    library.convnd_hip_delta_backward_workspace_size.restype = sz
    library.convnd_hip_delta_backward_workspace_size.argtypes = [ctypes.c_int, D, vp, vp, vp, vp]
    library.convnd_hip_delta_plan_describe.restype = ctypes.c_int
    library.convnd_hip_delta_plan_describe.argtypes = [ctypes.c_int, D, ctypes.c_int, ctypes.c_char_p, sz]
    library.convnd_hip_delta_backward.restype = ctypes.c_int
    library.convnd_hip_delta_backward.argtypes = [ctypes.c_int, D, *[vp] * 16, sz, vp]
    library.convnd_hip_linear_plan_describe.restype = ctypes.c_int
    library.convnd_hip_linear_plan_describe.argtypes = [ctypes.c_int, L, ctypes.c_int, ctypes.c_char_p, sz]
    library.convnd_hip_recurrence_plan_describe.restype = ctypes.c_int
    library.convnd_hip_recurrence_plan_describe.argtypes = [ctypes.c_int, R, ctypes.c_int, ctypes.c_char_p, sz]
    return library


KERNEL_IDS = {"forward_igemm": 0, "grad_input_igemm": 1, "grad_weight_mfma": 2}


def read_kernel_times(library):
    """{kernel name: (total ms, launches)} since the previous read (after a synchronize)."""
    out = {}
    for name, kid in KERNEL_IDS.items():
        total, count = ctypes.c_double(), ctypes.c_int64()
        if library.convnd_hip_timing_read(kid, ctypes.byref(total), ctypes.byref(count)) != SUCCESS:
            raise RuntimeError(library.convnd_hip_last_error().decode())
        out[name] = (total.value, count.value)
    return out


def dtype_code(dtype) -> int:
    import torch

    codes = {torch.float32: FLOAT32, torch.float64: FLOAT64, torch.float16: FLOAT16, torch.bfloat16: BFLOAT16}
    return codes[dtype]


def plan_names(library, x_shape, w_shape, stride, padding, dilation, groups, dtype):
    """(forward, input-gradient, weight-gradient) kernel families for a problem."""
    p = Problem.make(x_shape, w_shape, stride, padding, dilation, groups)
    code = dtype_code(dtype)
    return tuple(library.convnd_hip_plan_name(ctypes.byref(p), code, which).decode() for which in range(3))


def plan_details(library, x_shape, w_shape, stride, padding, dilation, groups, dtype):
    """Launch plans (forward, input gradient, weight gradient) as dicts."""
    import json

    p = Problem.make(x_shape, w_shape, stride, padding, dilation, groups)
    code = dtype_code(dtype)
    out = []
    for which in range(3):
        buffer = ctypes.create_string_buffer(1024)
        if library.convnd_hip_plan_describe(ctypes.byref(p), code, which, buffer, len(buffer)) != SUCCESS:
            raise RuntimeError(library.convnd_hip_last_error().decode())
        out.append(json.loads(buffer.value.decode()))
    return tuple(out)


def _described(library, describe, *args):
    import json

    buffer = ctypes.create_string_buffer(1024)
    if describe(*args, buffer, len(buffer)) != SUCCESS:
        raise RuntimeError(library.convnd_hip_last_error().decode())
    return json.loads(buffer.value.decode())


def linear_plan(library, rows, inputs, outputs, dtype, which=0):
    """Launch plan of a linear layer (0 forward, 1 and 2 one gradient, 3 both) as a dict."""
    p = LinearProblem(rows=rows, inputs=inputs, outputs=outputs, input_stride=inputs, grad_stride=outputs)
    return _described(library, library.convnd_hip_linear_plan_describe, dtype_code(dtype), ctypes.byref(p), which)


def recurrence_plan(library, batch, tokens, channels, dtype, backward=False):
    """Launch plan of a gated recurrence as a dict."""
    p = RecurrenceProblem(
        batch=batch, tokens=tokens, channels=channels, input_batch=tokens * channels, input_token=channels,
        gate_batch=tokens * channels, gate_token=channels,
    )
    describe = library.convnd_hip_recurrence_plan_describe
    return _described(library, describe, dtype_code(dtype), ctypes.byref(p), int(backward))


def delta_plan(library, batch, tokens, key_heads, heads, key_size, value_size, dtype, saving=False):
    """Launch plan of a gated delta rule as a dict."""
    p = DeltaProblem.make(batch, tokens, key_heads, heads, key_size, value_size, FLOAT32)
    describe = library.convnd_hip_delta_plan_describe
    return _described(library, describe, dtype_code(dtype), ctypes.byref(p), int(saving))
