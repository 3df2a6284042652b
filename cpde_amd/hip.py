"""ctypes binding of the device library's C ABI (include/cpde_hip.h).

Tests and the benchmark drive the kernels through exactly the entry points the
protocol server uses.  Loading fails loudly when the library is not built: there
is no CPU fallback.
"""
from __future__ import annotations

import ctypes
from pathlib import Path

import numpy as np

LIB_PATH = Path(__file__).resolve().parent / 'lib' / 'libcpde_hip.so'
HEADER = Path(__file__).resolve().parents[1] / 'include' / 'cpde_hip.h'

OK, EINVAL, EDEVICE, ECOMPILE = 0, 1, 2, 4


class CostStats(ctypes.Structure):
    _fields_ = [('value', ctypes.c_double), ('bad_sample', ctypes.c_int32), ('bad_component', ctypes.c_int32)]


class GradientStats(ctypes.Structure):
    _fields_ = [('squared_norm', ctypes.c_double), ('max_abs', ctypes.c_double),
                ('nonfinite_count', ctypes.c_uint64), ('first_nonfinite', ctypes.c_int32), ('pad_', ctypes.c_int32)]


_type_names = {}


def _type_name(dtype):
    name = _type_names.get(dtype)
    if name is None:
        name = _type_names[dtype] = str(dtype).rpartition('.')[2]
    return name


def _held(tensor):
    """(element type, GPU, sizes...) of a tensor."""
    if tensor.device.type == 'cpu':
        raise ValueError('the tensor is not on a GPU')
    return (_type_name(tensor.dtype), tensor.get_device(), *tensor.shape)


def _holds(name, view, want):
    """Refuses the view of a tensor of another type or GPU than `want`, or of less than its sizes."""
    held = view.held if view is not None else None
    if held != want and held is not None:  # (None: of an address)
        if held[:2] != want[:2]:
            raise ValueError(f'{name} is a tensor of {held[0]} on GPU {held[1]}, not of {want[0]} on GPU {want[1]}')
        if any(h < w for h, w in zip(held[2:], want[2:])):
            raise ValueError(f'{name} has the sizes {held[2:]}, less than {want[2:]}')


def _list_holds(name, a, kind, gpu, count):
    """The same of a list of `count` elements: a tensor, a Buffer by its bytes, or an address."""
    dtype = getattr(a, 'dtype', None)
    if dtype is None:
        if isinstance(a, Buffer) and a.nbytes < count * {'int64': 8, 'float16': 2, 'bfloat16': 2}.get(kind, 4):
            raise ValueError(f'{name} has {a.nbytes} bytes, not {count} of {kind}')
    elif _type_name(dtype) != kind or a.get_device() != gpu:
        raise ValueError(f'{name} is a tensor of {_type_name(dtype)} on {a.device}, not of {kind} on GPU {gpu}')
    elif a.numel() < count or not a.is_contiguous():
        raise ValueError(f'{name} is not {count} elements in a row')


class Heads(ctypes.Structure):
    """cpde_heads: a device tensor [batch][token][head][head_dim] by its element
    strides, the last axis contiguous.  A view made by `of` keeps the tensor's type and
    sizes, which calls check."""
    _fields_ = [('data', ctypes.c_void_p), ('batch', ctypes.c_int64), ('token', ctypes.c_int64),
                ('head', ctypes.c_int64)]
    held = None

    @classmethod
    def of(cls, tensor):
        """The view of a tensor on a GPU (torch's), which the caller keeps."""
        batch, token, head, last = tensor.stride()
        if last != 1 and tensor.shape[-1] > 1:
            raise ValueError('the last axis is not contiguous')
        view = cls(tensor.data_ptr(), batch, token, head)
        view.held = _held(tensor)
        return view


class Rows(ctypes.Structure):
    """cpde_rows: a device matrix by its row stride in elements, columns contiguous.  A
    view made by `of` keeps the tensor's type and sizes, which calls check."""
    _fields_ = [('data', ctypes.c_void_p), ('stride', ctypes.c_int64)]
    held = None

    @classmethod
    def of(cls, tensor):
        stride, last = tensor.stride()
        if last != 1 and tensor.shape[-1] > 1:
            raise ValueError('the last axis is not contiguous')
        view = cls(tensor.data_ptr(), stride)
        view.held = _held(tensor)
        return view


class Matrices(ctypes.Structure):
    """cpde_matrices: matrices [count][rows][columns] on a device by their element strides,
    columns contiguous.  A view made by `of` keeps the tensor's type and sizes, which calls
    check."""
    _fields_ = [('data', ctypes.c_void_p), ('matrix', ctypes.c_int64), ('row', ctypes.c_int64)]
    held = None

    @classmethod
    def of(cls, tensor):
        matrix, row, last = tensor.stride()
        if last != 1 and tensor.shape[-1] > 1:
            raise ValueError('the last axis is not contiguous')
        view = cls(tensor.data_ptr(), matrix, row)
        view.held = _held(tensor)
        return view


class AttentionShape(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in ('dtype', 'batch', 'query_tokens', 'key_tokens', 'heads', 'kv_heads',
                                              'head_dim', 'left', 'right', 'backward')] + [('scale', ctypes.c_float)]


class RotationShape(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in ('dtype', 'batch', 'tokens', 'heads', 'kv_heads', 'head_dim', 'rotated',
                                              'interleaved', 'norm', 'backward')] + \
               [('eps', ctypes.c_float), ('base', ctypes.c_double)]


class CpdeError(RuntimeError):
    def __init__(self, code, message):
        super().__init__(f'[{code}] {message}')
        self.code = code


_lib = None
vp = ctypes.c_void_p
i32 = ctypes.c_int
f32 = ctypes.c_float
i64 = ctypes.c_int64
u64 = ctypes.c_uint64
heads_p = ctypes.POINTER(Heads)
rows_p = ctypes.POINTER(Rows)
matrices_p = ctypes.POINTER(Matrices)

F32, F16, BF16 = 0, 1, 2    # element types of the operators on sequences
_element = ('float32', 'float16', 'bfloat16')
NONE, SIGMOID, RELU, SILU, GELU = range(5)    # activations

SIGNATURES = {
    'cpde_last_error': (ctypes.c_char_p, []),
    'cpde_device_open': (i32, [i32, ctypes.POINTER(vp)]),
    'cpde_device_open_on': (i32, [i32, vp, ctypes.POINTER(vp)]),
    'cpde_device_close': (i32, [vp]),
    'cpde_device_synchronize': (i32, [vp]),
    'cpde_device_info': (i32, [vp, ctypes.c_char_p, ctypes.c_size_t, ctypes.POINTER(i32)]),
    'cpde_buffer_alloc': (i32, [vp, ctypes.c_size_t, ctypes.POINTER(vp)]),
    'cpde_buffer_free': (i32, [vp, vp]),
    'cpde_buffer_upload': (i32, [vp, vp, vp, ctypes.c_size_t]),
    'cpde_buffer_download': (i32, [vp, vp, vp, ctypes.c_size_t]),
    'cpde_buffer_copy': (i32, [vp, vp, vp, ctypes.c_size_t]),
    'cpde_net_create': (i32, [vp, i32, vp, vp, vp, ctypes.POINTER(vp)]),
    'cpde_net_destroy': (i32, [vp]),
    'cpde_net_read': (i32, [vp, i32, i32, vp]),
    'cpde_net_write': (i32, [vp, i32, i32, vp]),
    'cpde_net_state': (i32, [vp, i32, i32, ctypes.POINTER(vp), ctypes.POINTER(i32)]),
    'cpde_net_active': (i32, [vp, i32]),
    'cpde_net_set_active': (i32, [vp, i32, i32]),
    'cpde_net_generation': (ctypes.c_uint64, [vp]),
    'cpde_plan_create': (i32, [vp, i32, i32, vp, i32, i32, ctypes.POINTER(vp)]),
    'cpde_plan_destroy': (i32, [vp]),
    'cpde_plan_stack': (i32, [vp, i32, i32, ctypes.POINTER(vp)]),
    'cpde_plan_stack_scale': (i32, [vp, i32, i32, vp]),
    'cpde_stacks_create': (i32, [vp, ctypes.POINTER(vp)]),
    'cpde_plan_bind': (i32, [vp, vp]),
    'cpde_stacks_destroy': (i32, [vp]),
    'cpde_activate': (i32, [vp, vp, i32, vp, i32, i32]),
    'cpde_forward': (i32, [vp]),
    'cpde_output': (i32, [vp, vp, i32, vp, i32, i32]),
    'cpde_gradients_defer': (i32, [vp, i32]),
    'cpde_costs_begin': (i32, [vp, i32]),
    'cpde_cost_matching': (i32, [vp, vp, i32, vp, vp, i32, i32, i32, i32, i32, i32]),
    'cpde_cost_polynomial': (i32, [vp, vp, i32, vp, vp, vp, i32, i32, i32, i32, i32, i32, i32]),
    'cpde_scale_adjoint': (i32, [vp, vp]),
    'cpde_backward': (i32, [vp, i32]),
    'cpde_inspect_gradients': (i32, [vp]),
    'cpde_epoch_matching': (i32, [vp, vp, i32, vp, vp, i32, i32, i32, i32, i32, i32]),
    'cpde_epoch_matching_static': (i32, [vp, vp, i32, vp, vp, i32, i32, i32, i32, i32, i32]),
    'cpde_epoch_matching_rprop': (i32, [vp, vp, i32, vp, vp, i32, i32, i32, i32, i32, i32]),
    'cpde_scalars_download': (i32, [vp, i32, vp, i32, vp]),
    'cpde_scalars_download_graph': (i32, [vp, i32, vp, i32, vp, vp, vp]),
    'cpde_rprop': (i32, [vp]),
    'cpde_scalars_download_rprop': (i32, [vp, i32, vp, i32, vp, vp, vp, vp]),
    'cpde_update_issue': (i32, [vp, i32, i32, i32, vp, i32, i32, f32]),
    'cpde_inspect_update_issue': (i32, [vp, i32, i32, i32, vp, i32, i32, f32, i32]),
    'cpde_update_resolve': (i32, [vp, vp, vp, vp, vp]),
    'cpde_gradients_discard': (i32, [vp]),
    'cpde_adam': (i32, [vp, i32, f32]),
    'cpde_set_steps': (i32, [vp, f32]),
    'cpde_restore_steps': (i32, [vp, f32]),
    'cpde_zero_gradient': (i32, [vp]),
    'cpde_reset_optimizer': (i32, [vp]),
    'cpde_program_compile': (i32, [vp, ctypes.c_char_p, ctypes.POINTER(vp), ctypes.c_char_p, ctypes.c_size_t]),
    'cpde_program_destroy': (i32, [vp]),
    'cpde_cost_expression': (i32, [vp, vp, vp, vp, i32, i32, i32, vp, vp, i32, i32, i32]),
    'cpde_epoch_expression': (i32, [vp, vp, vp, vp, i32, i32, i32, vp, vp, i32, i32, i32]),
    'cpde_attention_create': (i32, [vp, ctypes.POINTER(AttentionShape), ctypes.POINTER(vp)]),
    'cpde_attention_destroy': (i32, [vp]),
    'cpde_attention_info': (i32, [vp, ctypes.c_char_p, ctypes.c_size_t]),
    'cpde_attention_forward': (i32, [vp, heads_p, heads_p, heads_p, heads_p, vp, vp, vp]),
    'cpde_attention_backward': (i32, [vp, heads_p, heads_p, heads_p, heads_p, vp, heads_p, heads_p, heads_p, heads_p,
                                      vp, vp]),
    'cpde_embedding_create': (i32, [vp, i32, i32, i32, i64, i32, ctypes.POINTER(vp)]),
    'cpde_embedding_destroy': (i32, [vp]),
    'cpde_embedding_forward': (i32, [vp, vp, i64, rows_p, f32, rows_p]),
    'cpde_embedding_backward': (i32, [vp, vp, i64, rows_p, f32, rows_p, i32]),
    'cpde_dropout': (i32, [vp, i32, i64, i64, rows_p, rows_p, rows_p, ctypes.c_double, u64, u64]),
    'cpde_linear_create': (i32, [vp, i32, i64, i32, i32, i32, i32, ctypes.POINTER(vp)]),
    'cpde_linear_destroy': (i32, [vp]),
    'cpde_linear_info': (i32, [vp, i64, i32, ctypes.c_char_p, ctypes.c_size_t]),
    'cpde_linear_forward': (i32, [vp, i64, rows_p, rows_p, vp, rows_p, rows_p, rows_p]),
    'cpde_linear_backward': (i32, [vp, i64, rows_p, rows_p, rows_p, rows_p, rows_p, rows_p, vp, i32]),
    'cpde_rotation_create': (i32, [vp, ctypes.POINTER(RotationShape), ctypes.POINTER(vp)]),
    'cpde_rotation_destroy': (i32, [vp]),
    'cpde_rotation_forward': (i32, [vp, heads_p, heads_p, vp, vp, vp, heads_p, heads_p]),
    'cpde_rotation_backward': (i32, [vp, heads_p, heads_p, vp, vp, vp, heads_p, heads_p, heads_p, heads_p, vp, vp]),
    'cpde_orthogonal_create': (i32, [vp, i32, i32, i32, i32, i32, ctypes.POINTER(vp)]),
    'cpde_orthogonal_destroy': (i32, [vp]),
    'cpde_orthogonal_forward': (i32, [vp, matrices_p, matrices_p]),
    'cpde_orthogonal_update': (i32, [vp, matrices_p, matrices_p, matrices_p, f32, f32, f32, i32]),
    'cpde_capture_begin': (i32, [vp]),
    'cpde_capture_end': (i32, [vp, i32, vp]),
    'cpde_replay_launch': (i32, [vp]),
    'cpde_replay_destroy': (i32, [vp]),
    'cpde_epoch_expression_fused': (i32, [vp, vp, vp]),
    'cpde_graph_execute': (i32, [vp, vp, i32, i32, i32, vp, vp, vp, vp, vp, i32]),
    'cpde_jit_prepare': (i32, [i32, i32, vp, i32, vp, i32, i32, ctypes.c_char_p, ctypes.c_char_p, ctypes.c_size_t]),
    'cpde_trace_enable': (i32, [vp, i32]),
    'cpde_trace_read': (i32, [vp, i32, ctypes.POINTER(ctypes.c_uint64), ctypes.POINTER(ctypes.c_double),
                              ctypes.POINTER(ctypes.c_double)]),
    'cpde_trace_name': (ctypes.c_char_p, [i32]),
    'cpde_trace_kinds': (i32, []),
    'cpde_mark': (i32, [vp, i32]),
    'cpde_elapsed': (i32, [vp, i32, i32, ctypes.POINTER(f32)]),
}


def header_symbols():
    """Function names declared in include/cpde_hip.h."""
    import re
    text = HEADER.read_text()
    return sorted(set(re.findall(r'^\s*(?:int|uint64_t|const char\*)\s+(cpde_\w+)\s*\(', text, re.M)))


def load(path=None):
    global _lib
    if _lib is not None and path is None:
        return _lib
    p = Path(path) if path else LIB_PATH
    if not p.exists():
        raise RuntimeError(f'{p} is not built; run python -m cpde_amd.build')
    lib = ctypes.CDLL(str(p))
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args
    if path is None:
        _lib = lib
    return lib


def check(code):
    if code != OK:
        raise CpdeError(code, load().cpde_last_error().decode('utf-8', 'replace'))


def _ptr(a):
    return ctypes.c_void_p(a.ctypes.data)


def _address(a):
    """The device address of a Buffer, a tensor with data_ptr() (torch's), a pointer, or None."""
    if a is None or isinstance(a, (int, ctypes.c_void_p)):
        return a
    return a.ptr if isinstance(a, Buffer) else a.data_ptr()


class Buffer:
    """A device allocation (bytes); upload/download take numpy arrays."""

    def __init__(self, device, nbytes):
        self.device, self.nbytes = device, int(nbytes)
        p = vp()
        check(load().cpde_buffer_alloc(device.handle, self.nbytes, ctypes.byref(p)))
        self.ptr = p

    @classmethod
    def of(cls, device, array):
        a = np.ascontiguousarray(array)
        b = cls(device, max(a.nbytes, 4))
        b.upload(a)
        return b

    def upload(self, array):
        a = np.ascontiguousarray(array)
        assert a.nbytes <= self.nbytes
        check(load().cpde_buffer_upload(self.device.handle, self.ptr, _ptr(a), a.nbytes))

    def download(self, dtype, count):
        a = np.empty(count, dtype)
        check(load().cpde_buffer_download(self.device.handle, _ptr(a), self.ptr, a.nbytes))
        return a

    def free(self):
        if self.ptr:
            check(load().cpde_buffer_free(self.device.handle, self.ptr))
            self.ptr = None


class Device:
    """An open GPU.  stream: None for a stream of the library's own, or the handle
    of one of the caller's (0: the default stream), so that the library's work is
    in order with what else runs there."""

    def __init__(self, ordinal=0, stream=None):
        h = vp()
        if stream is None:
            check(load().cpde_device_open(ordinal, ctypes.byref(h)))
        else:
            check(load().cpde_device_open_on(ordinal, stream, ctypes.byref(h)))
        self.handle, self.ordinal = h, ordinal

    def info(self):
        name = ctypes.create_string_buffer(256)
        cu = i32()
        check(load().cpde_device_info(self.handle, name, 256, ctypes.byref(cu)))
        return name.value.decode(), cu.value

    def synchronize(self):
        check(load().cpde_device_synchronize(self.handle))

    def download_ptr(self, ptr, dtype, count):
        a = np.empty(count, dtype)
        check(load().cpde_buffer_download(self.handle, _ptr(a), ptr, a.nbytes))
        return a

    def upload_ptr(self, ptr, array):
        a = np.ascontiguousarray(array)
        check(load().cpde_buffer_upload(self.handle, ptr, _ptr(a), a.nbytes))

    def costs_begin(self, n):
        check(load().cpde_costs_begin(self.handle, n))

    def scalars(self, costs, layers):
        c = (CostStats * max(costs, 1))()
        g = (GradientStats * max(layers, 1))()
        check(load().cpde_scalars_download(self.handle, costs, ctypes.cast(c, vp), layers, ctypes.cast(g, vp)))
        return list(c)[:costs], list(g)[:layers]

    def mark(self, slot):
        check(load().cpde_mark(self.handle, slot))

    def elapsed(self, a, b):
        ms = f32()
        check(load().cpde_elapsed(self.handle, a, b, ctypes.byref(ms)))
        return ms.value

    def trace(self, on):
        check(load().cpde_trace_enable(self.handle, int(on)))

    def trace_report(self):
        """{kernel class: (launches, total device ms, total algorithmic work)}."""
        out = {}
        lib = load()
        for k in range(lib.cpde_trace_kinds()):
            n, ms, work = ctypes.c_uint64(), ctypes.c_double(), ctypes.c_double()
            check(lib.cpde_trace_read(self.handle, k, ctypes.byref(n), ctypes.byref(ms), ctypes.byref(work)))
            if n.value:
                out[lib.cpde_trace_name(k).decode()] = (n.value, ms.value, work.value)
        return out

    def dropout(self, dtype, rows, columns, x, y, probability, seed, offset=0, residual=None):
        """y = dropout(x) (+ residual), Rows of one type; the gradient is the same
        call on y's gradient with the same probability, seed and offset."""
        if 0 <= dtype < len(_element):
            want = (_element[dtype], self.ordinal, rows, columns)
            if x and x.held != want:
                _holds('x', x, want)
            if y and y.held != want:
                _holds('y', y, want)
            if residual and residual.held != want:
                _holds('residual', residual, want)
        check(load().cpde_dropout(self.handle, dtype, rows, columns, x, residual, y, probability, seed, offset))

    def capture_begin(self):
        check(load().cpde_capture_begin(self.handle))

    def capture_end(self, keep=True):
        """End the open capture; with `keep`, a Replay of it (already run once)."""
        h = vp()
        check(load().cpde_capture_end(self.handle, int(keep), ctypes.byref(h) if keep else None))
        return Replay(self, h) if keep else None

    def close(self):
        if self.handle:
            check(load().cpde_device_close(self.handle))
            self.handle = None


class Replay:
    """A recorded sequence of launches (cpde_capture_end)."""

    def __init__(self, device, handle):
        self.device, self.handle = device, handle

    def launch(self):
        check(load().cpde_replay_launch(self.handle))

    def destroy(self):
        if self.handle:
            check(load().cpde_replay_destroy(self.handle))
            self.handle = None


class Net:
    def __init__(self, device, neurons, linear, weights=None):
        self.device, self.neurons, self.linear = device, list(neurons), list(linear)
        n = np.asarray(neurons, np.int32)
        l = np.asarray(linear, np.int32)
        self._keep = [np.ascontiguousarray(w, np.float32) for w in weights] if weights is not None else None
        arr = None
        if self._keep is not None:
            P = ctypes.c_void_p * len(self._keep)
            arr = P(*[w.ctypes.data for w in self._keep])
        h = vp()
        check(load().cpde_net_create(device.handle, len(neurons), _ptr(n), _ptr(l),
                                     ctypes.cast(arr, vp) if arr is not None else None, ctypes.byref(h)))
        self.handle = h

    def state_ptr(self, t, b):
        p, c = vp(), i32()
        check(load().cpde_net_state(self.handle, t, b, ctypes.byref(p), ctypes.byref(c)))
        return p, c.value

    def _count(self, t, b):
        if not 0 <= t < len(self.neurons) - 1:
            self.state_ptr(t, b)   # the library's refusal
        return self.neurons[t + 1] * (self.neurons[t] + 1)

    def state(self, t, b):
        v = np.empty(self._count(t, b), np.float32)
        check(load().cpde_net_read(self.handle, t, b, _ptr(v)))
        return v

    def set_state(self, t, b, values):
        v = np.ascontiguousarray(values, np.float32)
        assert v.size == self._count(t, b)
        check(load().cpde_net_write(self.handle, t, b, _ptr(v)))

    def active(self, t):
        return load().cpde_net_active(self.handle, t)

    def gradient(self, t):
        return self.state(t, self.active(t))

    def rprop(self):
        check(load().cpde_rprop(self.handle))

    def download_rprop(self, costs):
        """The scalar download with RPROP behind it (no graph): cost and
        gradient totals, and whether the update applied."""
        layers = len(self.neurons) - 1
        c = (CostStats * max(costs, 1))()
        g = (GradientStats * layers)()
        updated = i32()
        check(load().cpde_scalars_download_rprop(self.device.handle, costs, ctypes.cast(c, vp), layers,
                                                 ctypes.cast(g, vp), None, self.handle, ctypes.byref(updated)))
        return list(c)[:costs], list(g), updated.value

    def issue_update(self, costs=0, method=0, step=0, lr=0.0, inspect=None):
        """cpde_update_issue (no graph); with `inspect` ('full' or 'short'),
        cpde_inspect_update_issue: the gradient statistics taken first, or the
        update launch's own finiteness test where the network allows."""
        layers = len(self.neurons) - 1
        if inspect is None:
            check(load().cpde_update_issue(self.device.handle, costs, layers, 0, self.handle, method, step, lr))
        else:
            check(load().cpde_inspect_update_issue(self.device.handle, costs, layers, 0, self.handle, method, step, lr,
                                                   int(inspect == 'full')))

    def resolve_update(self, costs=0):
        """cpde_update_resolve: cost and gradient totals, and whether the update applied."""
        layers = len(self.neurons) - 1
        c = (CostStats * max(costs, 1))()
        g = (GradientStats * layers)()
        updated = i32()
        check(load().cpde_update_resolve(self.device.handle, ctypes.cast(c, vp), ctypes.cast(g, vp), None,
                                         ctypes.byref(updated)))
        return list(c)[:costs], list(g), updated.value

    def adam(self, step, lr):
        check(load().cpde_adam(self.handle, step, lr))

    def set_steps(self, v):
        check(load().cpde_set_steps(self.handle, v))

    def restore_steps(self, v):
        check(load().cpde_restore_steps(self.handle, v))

    def inspect_gradients(self):
        check(load().cpde_inspect_gradients(self.handle))

    def destroy(self):
        if self.handle:
            check(load().cpde_net_destroy(self.handle))
            self.handle = None


class Plan:
    def __init__(self, net, table, width, backward=True):
        self.net, self.width = net, width
        self.table = np.ascontiguousarray(table, np.int32)
        self.rows = self.table.shape[0]
        h = vp()
        check(load().cpde_plan_create(net.handle, self.rows, self.table.shape[1] - 1, _ptr(self.table), width,
                                      int(backward), ctypes.byref(h)))
        self.handle = h

    def stack_ptr(self, layer, kind):
        p = vp()
        check(load().cpde_plan_stack(self.handle, layer, kind, ctypes.byref(p)))
        return p

    def stack(self, layer, kind):
        """(width, rows, n) float32 view of a stack."""
        n = self.net.neurons[layer]
        a = self.net.device.download_ptr(self.stack_ptr(layer, kind), np.float32, self.width * self.rows * n)
        return a.reshape(self.width, self.rows, n)

    def stack_scale(self, layer, kind):
        """(rows,) factors turning stored rows of a stack into unscaled rows."""
        f = np.zeros(self.rows, np.float32)
        check(load().cpde_plan_stack_scale(self.handle, layer, kind, _ptr(f)))
        return f

    def unscaled_stack(self, layer, kind):
        """stack() with every row in the reference's (unscaled) form."""
        return self.stack(layer, kind) * self.stack_scale(layer, kind)[None, :, None]

    def set_stack(self, layer, kind, values):
        self.net.device.upload_ptr(self.stack_ptr(layer, kind), np.ascontiguousarray(values, np.float32))

    def activate(self, data_buffer, data_width, rows, offset, valid):
        r = np.ascontiguousarray(rows, np.int32)
        check(load().cpde_activate(self.handle, data_buffer.ptr, data_width, _ptr(r), offset, valid))

    def forward(self):
        check(load().cpde_forward(self.handle))

    def backward(self, accumulate=False):
        check(load().cpde_backward(self.handle, int(accumulate)))

    def output(self, dest_buffer, dest_width, rows, offset, valid):
        r = np.ascontiguousarray(rows, np.int32)
        check(load().cpde_output(self.handle, dest_buffer.ptr, dest_width, _ptr(r), offset, valid))

    def epoch_matching(self, target, target_width, target_rows, weights, weight_samples, offset, valid, cost_index,
                       collect=True, accumulate=False):
        """forward + matching cost + backward of the activated chunk in one pass."""
        check(load().cpde_epoch_matching(self.handle, target.ptr, target_width, target_rows.ptr, weights.ptr,
                                         weight_samples, offset, valid, cost_index, int(collect), int(accumulate)))

    def epoch_matching_rprop(self, target, target_width, target_rows, weights, weight_samples, offset, valid,
                             cost_index, collect=True, accumulate=False):
        """epoch_matching, then RPROP on the network, the update riding in the
        gradient reduction's launch."""
        check(load().cpde_epoch_matching_rprop(self.handle, target.ptr, target_width, target_rows.ptr, weights.ptr,
                                               weight_samples, offset, valid, cost_index, int(collect),
                                               int(accumulate)))

    def epoch_matching_static(self, target, target_width, target_rows, weights, weight_samples, offset, valid,
                              cost_index, collect=True, accumulate=False):
        """epoch_matching with the library's static scratch: no allocation."""
        check(load().cpde_epoch_matching_static(self.handle, target.ptr, target_width, target_rows.ptr, weights.ptr,
                                                weight_samples, offset, valid, cost_index, int(collect),
                                                int(accumulate)))

    def matching(self, target, target_width, target_rows, weights, weight_samples, offset, valid, cost_index,
                 collect=True, gradient=True):
        check(load().cpde_cost_matching(self.handle, target.ptr, target_width, target_rows.ptr, weights.ptr,
                                        weight_samples, offset, valid, cost_index, int(collect), int(gradient)))

    def destroy(self):
        if self.handle:
            check(load().cpde_plan_destroy(self.handle))
            self.handle = None


class Attention:
    """Attention of one shape and type (cpde_attention_shape).  Tensors are Heads,
    lse and the lengths device addresses (or tensors, or Buffers)."""

    def __init__(self, device, dtype, batch, query_tokens, key_tokens, heads, kv_heads, head_dim, scale=0.0, left=-1,
                 right=-1, backward=True):
        self.device = device
        shape = AttentionShape(dtype, batch, query_tokens, key_tokens, heads, kv_heads, head_dim, left, right,
                               int(backward), scale)
        h = vp()
        check(load().cpde_attention_create(device.handle, ctypes.byref(shape), ctypes.byref(h)))
        self.handle = h
        self.query_side = (_element[dtype], device.ordinal, batch, query_tokens, heads, head_dim)
        self.key_side = (_element[dtype], device.ordinal, batch, key_tokens, kv_heads, head_dim)
        self.batch, self.rows = batch, batch * heads * query_tokens

    def info(self):
        """The kernels that the calls run, and over how many splits."""
        text = ctypes.create_string_buffer(256)
        check(load().cpde_attention_info(self.handle, text, 256))
        return text.value.decode()

    def _check(self, queries, keys, lse, query_lengths, key_lengths):
        """Tensors on the queries' and the keys' side, by name, and lists."""
        for name, view in queries.items():
            _holds(name, view, self.query_side)
        for name, view in keys.items():
            _holds(name, view, self.key_side)
        gpu = self.query_side[1]
        if lse is not None:
            _list_holds('lse', lse, 'float32', gpu, self.rows)
        if query_lengths is not None:
            _list_holds('query_lengths', query_lengths, 'int32', gpu, self.batch)
        if key_lengths is not None:
            _list_holds('key_lengths', key_lengths, 'int32', gpu, self.batch)

    def forward(self, q, k, v, out, lse=None, query_lengths=None, key_lengths=None):
        self._check({'q': q, 'out': out}, {'k': k, 'v': v}, lse, query_lengths, key_lengths)
        check(load().cpde_attention_forward(self.handle, q, k, v, out, _address(lse), _address(query_lengths),
                                            _address(key_lengths)))

    def backward(self, q, k, v, out, lse, dout, dq, dk, dv, query_lengths=None, key_lengths=None):
        self._check({'q': q, 'out': out, 'dout': dout, 'dq': dq}, {'k': k, 'v': v, 'dk': dk, 'dv': dv}, lse, query_lengths,
                    key_lengths)
        check(load().cpde_attention_backward(self.handle, q, k, v, out, _address(lse), dout, dq, dk, dv,
                                             _address(query_lengths), _address(key_lengths)))

    def destroy(self):
        if self.handle:
            check(load().cpde_attention_destroy(self.handle))
            self.handle = None


class Embedding:
    """Lookups of at most `tokens` ids a call in a table of rows x width, and the
    table's gradient.  ids are a device address (or tensor, or Buffer), the others Rows."""

    def __init__(self, device, dtype, rows, width, tokens, index_bytes=4):
        self.device = device
        h = vp()
        check(load().cpde_embedding_create(device.handle, dtype, rows, width, tokens, index_bytes, ctypes.byref(h)))
        self.handle = h
        self.element, self.rows, self.width, self.tokens = _element[dtype], rows, width, tokens
        self.index = 'int64' if index_bytes == 8 else 'int32'

    def _check(self, ids, tokens, names, table, table_type, rows):
        if tokens > self.tokens:
            return  # (the library refuses it)
        gpu = self.device.ordinal
        if ids is not None:
            _list_holds('ids', ids, self.index, gpu, tokens)
        _holds(names[0], table, (table_type, gpu, self.rows, self.width))
        _holds(names[1], rows, (self.element, gpu, tokens, self.width))

    def forward(self, ids, tokens, table, out, scale=1.0):
        self._check(ids, tokens, ('table', 'out'), table, self.element, out)
        check(load().cpde_embedding_forward(self.handle, _address(ids), tokens, table, scale, out))

    def backward(self, ids, tokens, dout, dtable, scale=1.0, accumulate=False):
        self._check(ids, tokens, ('dtable', 'dout'), dtable, 'float32', dout)
        check(load().cpde_embedding_backward(self.handle, _address(ids), tokens, dout, scale, dtable, int(accumulate)))

    def destroy(self):
        if self.handle:
            check(load().cpde_embedding_destroy(self.handle))
            self.handle = None


class Linear:
    """y = activation(x W^T + bias) + residual of at most `rows` rows a call, and its
    gradient; W is [outputs][inputs].  Matrices are Rows, biases device addresses (or
    tensors, or Buffers) of `outputs` values of the plan's type."""

    def __init__(self, device, dtype, rows, inputs, outputs, activation=NONE, backward=True):
        self.device = device
        h = vp()
        check(load().cpde_linear_create(device.handle, dtype, rows, inputs, outputs, activation, int(backward),
                                        ctypes.byref(h)))
        self.handle = h
        self.element, self.rows, self.inputs, self.outputs = _element[dtype], rows, inputs, outputs

    def _check(self, rows, inputs, outputs, weights, bias):
        """Matrices by name: as wide as the inputs, as the outputs, and of the weights' sizes."""
        if rows > self.rows:
            return  # (the library refuses it)
        gpu = self.device.ordinal
        for views, want in ((inputs, (rows, self.inputs)), (outputs, (rows, self.outputs)),
                            (weights, (self.outputs, self.inputs))):
            for name, view in views.items():
                _holds(name, view, (self.element, gpu, *want))
        for name, a in bias.items():
            if a is not None:
                _list_holds(name, a, self.element, gpu, self.outputs)

    def info(self, rows, aligned=True):
        """The kernels that calls of `rows` rows run on contiguous matrices (aligned: from whole
        16 bytes on), their tiles and splits."""
        text = ctypes.create_string_buffer(256)
        check(load().cpde_linear_info(self.handle, rows, int(aligned), text, 256))
        return text.value.decode()

    def forward(self, rows, x, weight, y, bias=None, residual=None, pre=None):
        self._check(rows, {'x': x}, {'y': y, 'residual': residual, 'pre': pre}, {'weight': weight}, {'bias': bias})
        check(load().cpde_linear_forward(self.handle, rows, x, weight, _address(bias), residual, y, pre))

    def backward(self, rows, x, weight, dy, pre=None, dx=None, dweight=None, dbias=None, accumulate=False):
        self._check(rows, {'x': x, 'dx': dx}, {'pre': pre, 'dy': dy}, {'weight': weight, 'dweight': dweight},
                    {'dbias': dbias})
        check(load().cpde_linear_backward(self.handle, rows, x, weight, pre, dy, dx, dweight, _address(dbias),
                                          int(accumulate)))

    def destroy(self):
        if self.handle:
            check(load().cpde_linear_destroy(self.handle))
            self.handle = None


class Rotation:
    """Each head's norm and its rotation by the token's position, of queries and keys
    (cpde_rotation_shape; rotated: None for whole heads), and their gradients.  Tensors are
    Heads, weights and positions device addresses (or tensors, or Buffers)."""

    def __init__(self, device, dtype, batch, tokens, heads, kv_heads, head_dim, rotated=None, interleaved=False,
                 base=10000.0, eps=1e-6, norm=True, backward=True):
        self.device = device
        shape = RotationShape(dtype, batch, tokens, heads, kv_heads, head_dim, head_dim if rotated is None else rotated,
                              int(interleaved), int(norm), int(backward), eps, base)
        h = vp()
        check(load().cpde_rotation_create(device.handle, ctypes.byref(shape), ctypes.byref(h)))
        self.handle = h
        gpu = device.ordinal
        self.query_side = (_element[dtype], gpu, batch, tokens, heads, head_dim)
        self.key_side = (_element[dtype], gpu, batch, tokens, kv_heads, head_dim)

    def _check(self, queries, keys, weights, positions):
        for views, want in ((queries, self.query_side), (keys, self.key_side)):
            for name, view in views.items():
                if want[4]:
                    _holds(name, view, want)
        element, gpu, batch, tokens, _, dim = self.query_side
        for name, a in weights.items():
            if a is not None:
                _list_holds(name, a, element, gpu, dim)
        if positions is not None:
            _list_holds('positions', positions, 'int32', gpu, batch * tokens)

    def forward(self, q, k, q_out, k_out, q_weight=None, k_weight=None, positions=None):
        self._check({'q': q, 'q_out': q_out}, {'k': k, 'k_out': k_out}, {'q_weight': q_weight, 'k_weight': k_weight}, positions)
        check(load().cpde_rotation_forward(self.handle, q, k, _address(q_weight), _address(k_weight), _address(positions),
                                           q_out, k_out))

    def backward(self, q, k, dq_out, dk_out, dq, dk, q_weight=None, k_weight=None, dq_weight=None, dk_weight=None,
                 positions=None):
        self._check({'q': q, 'dq_out': dq_out, 'dq': dq}, {'k': k, 'dk_out': dk_out, 'dk': dk},
                    {'q_weight': q_weight, 'k_weight': k_weight, 'dq_weight': dq_weight, 'dk_weight': dk_weight}, positions)
        check(load().cpde_rotation_backward(self.handle, q, k, _address(q_weight), _address(k_weight), _address(positions),
                                            dq_out, dk_out, dq, dk, _address(dq_weight), _address(dk_weight)))

    def destroy(self):
        if self.handle:
            check(load().cpde_rotation_destroy(self.handle))
            self.handle = None


class Orthogonal:
    """`count` matrices of rows x columns brought near the orthogonal ones of their singular
    vectors, and an optimizer's step along them.  Tensors are Matrices."""

    def __init__(self, device, dtype, count, rows, columns, steps=5):
        self.device = device
        h = vp()
        check(load().cpde_orthogonal_create(device.handle, dtype, count, rows, columns, steps, ctypes.byref(h)))
        self.handle = h
        self.side = (_element[dtype], device.ordinal, count, rows, columns)

    def forward(self, x, out):
        _holds('x', x, self.side)
        _holds('out', out, self.side)
        check(load().cpde_orthogonal_forward(self.handle, x, out))

    def update(self, gradient, momentum, weight, rate, momentum_factor=0.95, decay=0.0, nesterov=True):
        """One step of the weights, in place, and of their (float) momentum."""
        _holds('gradient', gradient, self.side)
        _holds('momentum', momentum, ('float32', *self.side[1:]))
        _holds('weight', weight, self.side)
        check(load().cpde_orthogonal_update(self.handle, gradient, momentum, weight, rate, momentum_factor, decay,
                                            int(nesterov)))

    def destroy(self):
        if self.handle:
            check(load().cpde_orthogonal_destroy(self.handle))
            self.handle = None


def jit_prepare(table, neurons, width=0, compute_units=256, arch='gfx950'):
    """Compile the fused kernels of (schema, architecture) for chunks of `width`
    points on a device of `compute_units` CUs into the code-object cache; no
    device needed.  Returns the compiler log."""
    t = np.ascontiguousarray(table, np.int32)
    n = np.ascontiguousarray(neurons, np.int32)
    log = ctypes.create_string_buffer(1 << 16)
    code = load().cpde_jit_prepare(t.shape[0], t.shape[1] - 1, _ptr(t), len(n), _ptr(n), width, compute_units,
                                   arch.encode(), log, len(log))
    if code != OK:
        raise CpdeError(code, load().cpde_last_error().decode('utf-8', 'replace') + log.value.decode())
    return log.value.decode()


def wire_to_stack(a):
    """(rows, channels, points) -> (points, rows, channels)."""
    return np.ascontiguousarray(np.asarray(a).transpose(2, 0, 1))


def stack_to_reference(s):
    """(points, rows, n) -> reference layout (rows, points, n)."""
    return np.ascontiguousarray(np.asarray(s).transpose(1, 0, 2))


class MatchingRun:
    """One matching cost on one plan: the unit of work of the benchmark step
    (forward + cost + weight gradient), driven through the C ABI."""

    def __init__(self, device, workload, chunk=None, one_pass=True, static_scratch=False):
        wl = workload
        self.device, self.wl = device, wl
        self.one_pass = one_pass
        self.static_scratch = static_scratch
        self.net = Net(device, wl.neurons, wl.linear, wl.init)
        self.samples = wl.size
        self.width = min(chunk or wl.chunk or wl.size, wl.size)
        self.plan = Plan(self.net, wl.cost_schema, self.width, True)
        # wire layouts: data [rows][samples][channels], weights [R][weight_samples][outputs]
        self.data = Buffer.of(device, np.ascontiguousarray(wl.inputs.transpose(0, 2, 1), np.float32))
        self.target = Buffer.of(device, np.ascontiguousarray(wl.target[:, :, None], np.float32))
        self.target_rows = Buffer.of(device, np.ascontiguousarray(wl.target_rows, np.int32))
        self.weights = Buffer.of(device, np.ascontiguousarray(wl.weight_block(), np.float32))
        self.weight_samples = wl.weight_samples
        self.rows = np.ascontiguousarray(wl.cost_rows, np.int32)
        self._loaded = None
        device.costs_begin(1)

    def step(self, collect=True, update=False):
        """forward + cost + backward over every chunk (Server::pass).  As in
        Server::activate (cuda/cpde_server.cu:163) the input copy is skipped when
        the loaded chunk is unchanged.  `update`: then RPROP, riding in the last
        chunk's gradient reduction (one-pass epochs) or launched after it."""
        self.device.costs_begin(1)
        first = True
        for offset in range(0, self.samples, self.width):
            valid = min(self.width, self.samples - offset)
            if self._loaded != (offset, valid):
                self.plan.activate(self.data, self.samples, self.rows, offset, valid)
                self._loaded = (offset, valid)
            last = offset + self.width >= self.samples
            cost = (self.target, self.samples, self.target_rows, self.weights, self.weight_samples, offset, valid, 0,
                    collect)
            if update and last and self.one_pass and not self.static_scratch:
                self.plan.epoch_matching_rprop(*cost, not first)
                return
            if self.static_scratch:
                self.plan.epoch_matching_static(*cost, not first)
            elif self.one_pass:
                self.plan.epoch_matching(*cost, not first)
            else:
                self.plan.forward()
                self.plan.matching(*cost, True)
                self.plan.backward(not first)
            first = False
        if update:
            self.net.rprop()

    def loss(self):
        c, _ = self.device.scalars(1, 0)
        return c[0].value

    def gradients(self):
        return [self.net.gradient(t) for t in range(len(self.wl.neurons) - 1)]

    def close(self):
        for b in (self.data, self.target, self.target_rows, self.weights):
            b.free()
        self.plan.destroy()
        self.net.destroy()
