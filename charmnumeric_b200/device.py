"""Arrays and the device memory of other libraries, through ``__cuda_array_interface__``."""
import numpy as np

from .frontend import _new_array, _normalize_dtype, _normalize_shape, execute


class DeviceView:
    """This rank's rows of an array where they are, for a library that reads
    ``__cuda_array_interface__``.  The interface names the stream the values are made on; a library
    that does not order itself behind it has to (``stream`` is its handle).  It shows the memory that the
    array has now: a stencil sweep, or a prompt with its state in place, moves an array to other memory."""

    def __init__(self, array, shape, pointer, stream):
        self.array = array  # keeps it from being released
        self.stream = stream
        self.__cuda_array_interface__ = {"shape": shape, "typestr": array.dtype.str, "data": (pointer, False),
                                         "strides": None, "version": 3, "stream": stream}


def device_view(array, interface):
    """View of a whole array's memory; everything recorded so far is executed (not waited for)."""
    execute(interface)
    info = interface.context.array_info(array.name)
    begin, end = info["rows"]
    pointer, stream = interface.context.device_array(array.name)
    return DeviceView(array, (end - begin,) + tuple(array.shape[1:]), pointer, stream)


def from_device(interface, source, stream=None):
    """A copy of another library's device array (dense, on the interface's GPU) as an ``Array``.  The copy
    is ordered behind ``stream``, the handle of the stream that the values are made on, and that stream
    behind the copy.  Without it the stream is the one that ``source`` names in its interface, or else the default
    stream: give it for tensors of libraries that name none and work on streams of their own (of torch's,
    ``torch.cuda.current_stream().cuda_stream``)."""
    about = getattr(source, "__cuda_array_interface__", None)
    if about is None:
        raise TypeError(f"{type(source).__name__} has no __cuda_array_interface__")
    shape = _normalize_shape(about["shape"])
    dtype = _normalize_dtype(np.dtype(about["typestr"]))
    strides = about.get("strides")
    if strides is not None:
        dense, step = [], dtype.itemsize
        for extent in reversed(shape):
            dense.insert(0, step)
            step *= extent
        if any(extent > 1 and a != b for extent, a, b in zip(shape, strides, dense)) and 0 not in shape:
            raise ValueError("from_device takes dense row-major arrays")
    if about.get("mask") is not None:
        raise ValueError("from_device takes no masked arrays")
    execute(interface)
    out = _new_array(shape, dtype)
    if 0 in shape:
        interface.context.put(out.name, np.empty(shape, dtype))
    else:
        interface.context.put_device(out.name, shape, dtype, about["data"][0], int(about.get("stream") or 0) if stream is None else int(stream))
    out._info.materialised = True
    if isinstance(source, DeviceView):
        out._info.set_group(source.array._info.group)
    return out
