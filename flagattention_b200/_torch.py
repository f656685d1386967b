"""torch helpers shared by the operator modules (device memory, streams)."""

import ctypes
import functools
import threading

import torch

from flagattention_b200 import _lib

_DTYPES = {torch.bfloat16: _lib.FA_DTYPE_BF16, torch.float16: _lib.FA_DTYPE_F16,
           torch.float32: _lib.FA_DTYPE_F32}


def dtype_code(t):
    try:
        return _DTYPES[t.dtype]
    except KeyError as e:
        raise _lib.InvalidArgument(f"unsupported dtype {t.dtype}") from e


def ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def stream_of(t):
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def raw_stream(device_index):
    """Handle of the device's current stream, as an integer (``stream_of``
    without building a Stream object: about 2 us less per call)."""
    return torch._C._cuda_getCurrentRawStream(device_index)


def current_device():
    """Index of the calling thread's current device: where the library launches
    (a call on another one enters its tensors' device first)."""
    return torch._C._cuda_getDevice()


def on_tensors_device(fn):
    """fn with the device of its first argument current during the call."""
    first = fn.__code__.co_varnames[0]

    @functools.wraps(fn)
    def call(*args, **kwargs):
        tensor = args[0] if args else kwargs.get(first)
        if not isinstance(tensor, torch.Tensor) or not tensor.is_cuda or \
                tensor.get_device() == current_device():
            return fn(*args, **kwargs)
        with torch.cuda.device(tensor.get_device()):
            return fn(*args, **kwargs)
    return call


_templates = {}


def empty(shape, dtype, device_index):
    """torch.empty on a GPU.  ``empty_like`` of a one-element tensor expanded to
    the shape costs 1.3 us on the host where ``torch.empty`` costs 2.4."""
    key = (shape, dtype, device_index)
    t = _templates.get(key)
    if t is None:
        device = torch.device("cuda", device_index)
        if 0 in shape:
            return torch.empty(shape, dtype=dtype, device=device)
        if len(_templates) >= 4096:
            _templates.clear()
        t = _templates[key] = torch.empty(1, dtype=dtype, device=device).expand(shape)
    return torch.empty_like(t, memory_format=torch.contiguous_format)


_workspaces = {}


def stream_workspace(size, device_index, stream):
    """Scratch of at least `size` bytes for one call on the given stream handle.

    Kept per stream and grown: the stream orders the calls that share it.  A
    call that is being captured gets its own, which lives as long as the graph.
    Returns (tensor to keep until the call is queued, address)."""
    if torch._C._cuda_isCurrentStreamCapturing():
        t = torch.empty(size, dtype=torch.uint8, device=torch.device("cuda", device_index))
        return t, t.data_ptr()
    held = _workspaces.get((device_index, stream))
    if held is None or held[2] < size:
        t = torch.empty(size, dtype=torch.uint8, device=torch.device("cuda", device_index))
        held = _workspaces[(device_index, stream)] = (t, t.data_ptr(), size)
    return held[0], held[1]


# held while a call's launches are queued: two threads on one stream must not
# interleave the two kernels that share a workspace
launch_lock = threading.Lock()


def require_cuda(*tensors):
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise _lib.InvalidArgument("flagattention_b200 operators take CUDA tensors only "
                                       "(there is no CPU path)")


def sm_count(device):
    n = ctypes.c_int32(0)
    _lib.check(_lib.lib().fa_device_sm_count(device.index if device.index is not None
                                             else torch.cuda.current_device(), ctypes.byref(n)),
               "fa_device_sm_count")
    return n.value


_status = {}


def status_word(device):
    """Per-device int32 the kernels set when a bounded wait gives up."""
    key = device.index if device.index is not None else torch.cuda.current_device()
    t = _status.get(key)
    if t is None:
        t = torch.zeros(1, dtype=torch.int32, device=device)
        _status[key] = t
    return t


_status_ptr = {}


def status_ptr(device_index):
    """Address of the device's status word."""
    p = _status_ptr.get(device_index)
    if p is None:
        p = _status_ptr[device_index] = status_word(torch.device("cuda", device_index)).data_ptr()
    return p


def read_status(device):
    """Synchronise and return (then clear) the device status word (0 = ok)."""
    t = status_word(device)
    v = int(t.item())
    if v:
        t.zero_()
    return v
