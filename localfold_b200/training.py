"""Operators for training and for 8-bit operands around the pair stack: LayerNorm with its gradients, activations kept in 8 bits, and the
projection on 8-bit operands with its gradients.  The reference runs the stack forward only: no counterpart there.

They stand beside the operators of ``operators.py`` and are called alike (``run(input[, options])`` on a ``Device``), but take
and return CUDA tensors only.  A call enqueues on the device's stream and returns.  Results and workspaces come from torch's
allocator, so a call can be captured into a CUDA graph (on the stream that the ``Device`` was made on) and graphs share nothing.  A device whose
stream is not torch's current one waits for the work enqueued there before it writes into such memory; its inputs are ordered as for
every operator (``Device``).  Gradients are calls of their own: autograd is not told of any, and results of tensors that require a gradient require none.

    norm, linear = lf.LayerNormGpu(dev), lf.Float8LinearGpu(dev)
    weights = lf.prepare_float8_linear_weights(dev, weight, bias)                 # [out][in], encoded once (update() after a step)
    a = norm.run({"rows": r, "channels": c, "activations": x, "scale": g, "offset": b}, {"checkpoint": "e4m3", "encode": "e4m3"})
    shape = {"rows": r, "channels": c, "outChannels": n}
    y = linear.run({**shape, "activations": a["output"], "weights": weights})["output"]
    back = linear.input_gradient({**shape, "gradient": dy, "weights": weights})
    grads = linear.weight_gradient({**shape, "gradient": dy, "activations": a["output"]})         # "weight", "bias"
    dx = norm.backward({"rows": r, "channels": c, "gradient": back["output"], "activations": a["checkpoint"], "mean": a["mean"],
                        "inverseDeviation": a["inverseDeviation"], "scale": g})                   # "activations", "scale", "offset"
"""
from __future__ import annotations

import struct
import sys
import weakref

import numpy as np

from . import _native as nat
from ._native import RangeError
from .operators import Device, EncodedTensor, _device, _positive, _torch_stream, _variance

_FORMAT = {"e4m3": nat.FLOAT8_E4M3, "e5m2": nat.FLOAT8_E5M2}
_DTYPE = {"f32": nat.DTYPE_F32, "bf16": nat.DTYPE_BF16}

# The descriptors (the ctypes structures of the same names), packed: small calls take a few microseconds, of which filling a structure
# field by field was one.  A matrix is its five fields.
_MATRIX = "qiiQQ"
_ENCODE = struct.Struct("@" + 2 * _MATRIX + "iiQ")
_DECODE = struct.Struct("@" + _MATRIX + "iiQ")
_LAYER_NORM = struct.Struct("@qiiif6Q" + 2 * _MATRIX)
_LAYER_NORM_BACKWARD = struct.Struct("@qiiQQ" + _MATRIX + "8Q")
_LINEAR = struct.Struct("@" + 2 * _MATRIX + "QiiQQQQ")
_WEIGHT_GRADIENT = struct.Struct("@" + _MATRIX + "Q" + _MATRIX + "ii4Q")
_NO_MATRIX = (0, 0, 0, 0, 0)
_NO_OPTIONS = {}
_MOST = 2 ** 31 - 1                                # rows and channels are 32-bit numbers in the kernels
_MOST_GRADIENT = 2 ** 22                           # channels of either side of a weight's gradient
_LARGEST = (2 - 2.0 ** -23) * 2.0 ** 127           # of float32
_AS_IT_WAS = object()


def _format(value, name="format"):
    if value not in _FORMAT:
        raise ValueError(f'{name} must be "e4m3" or "e5m2"; received {value!r}')
    return value


def _size(inp, name):
    value = inp[name]
    if type(value) is not int or not 0 < value <= _MOST:
        _positive(name, value)
        if value > _MOST:
            raise RangeError(f"{name} must be at most {_MOST}; received {value}")
        value = int(value)
    return value


_names = {}      # torch dtype -> "f32" | "bf16"
_Tensor = None   # torch.Tensor, with the first


def _torch():
    global _Tensor
    import torch
    if not _names:
        _Tensor = torch.Tensor
        _names.update({torch.float32: "f32", torch.bfloat16: "bf16"})
    return torch


def _has_memory(name, value):
    """A fake tensor passes every other check; the library would take it for one that was left out.  (One that a function transform has wrapped raises as soon as its
    address is asked for.)"""
    try:
        if value.data_ptr():
            return
    except RuntimeError:
        pass
    raise ValueError(f"{name} must be a tensor with memory of its own; received {type(value).__name__}")


def _tensor(device, name, value, count, only=None):
    """A tensor argument: on the device's GPU, contiguous, float32 or bfloat16 (``only``: one of them), of ``count`` values.
    Returns "f32" or "bf16"."""
    if getattr(value, "is_cuda", False) and value.get_device() == device.ordinal:
        dtype = _names.get(value.dtype)
        try:
            if dtype is not None and (only is None or only == dtype) and value.numel() == count and value.is_contiguous() and (type(value) is _Tensor or value.data_ptr()):
                return dtype
        except RuntimeError:      # (no address: below)
            pass
    if not getattr(value, "is_cuda", False):
        raise ValueError(f"{name} must be a CUDA tensor")
    if value.get_device() != device.ordinal:
        raise ValueError(f"{name} is on {value.device}, the device's GPU is cuda:{device.ordinal}")
    _torch()
    dtype = _names.get(value.dtype)
    if dtype is None or only not in (None, dtype):
        raise ValueError(f"{name} must be {only or 'f32 or bf16'}; received {value.dtype}")
    if not value.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if value.numel() != count:
        raise RangeError(f"{name} has {value.numel()} values; expected {count}")
    _has_memory(name, value)
    return dtype


def _torch_dtype(name):
    torch = _torch()
    return torch.float32 if name == "f32" else torch.bfloat16


def _capturing():
    torch = _torch()
    return torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()


def _call(device, function, desc, tensors, output=None, fresh=True, weights=None):
    """One library call and its result object.  Where torch's current stream is not the device's: a device with a stream of its own waits for
    torch's work first, and so does any device where the call has taken memory from torch's allocator (``fresh``), which torch's work may still
    be using for what it held before.  The device holds the call's tensors until its stream is done with them, so that torch does not
    give their memory away before."""
    current = _torch_stream(device.ordinal)
    if current != device.stream and _capturing():      # (the device's stream would run outside the graph, or be left in it)
        raise RuntimeError(f"a call is captured on its device's stream ({device.stream:#x}); torch's current stream ({current:#x}) is being captured: make the Device on it")
    if current != device.stream and (device._own_stream or fresh):
        device.check(device.lib.lf_context_await(device.handle, current))
    res = nat.Result()
    status = function(device.handle, desc, res)
    if status != nat.LF_OK:
        device.check(status)
    if current != device.stream:
        device.hold(tensors)
    elif weights is not None and weights._origin != current:
        weights._read_on(device)
    return {"output": output, "elapsedMilliseconds": 0.0, "memory": {"peakBytes": res.peak_bytes}, "launches": res.launches}


def _sizes(rows, channels):
    """Bytes of the codes and of the exponents (``lf_float8_code_bytes``, ``lf_float8_exponent_bytes``)."""
    return rows * ((channels + 15) & -16), ((channels + 511) >> 9) * ((rows + 127) >> 7) * 512


_empty = {}      # (GPU, dtype) -> an empty tensor: new memory of that kind takes least time from one


def _new(like, dtype, shape):
    key = (like.get_device(), dtype)
    proto = _empty.get(key)
    if proto is None:      # (a plain tensor, whatever the call's own are and whichever mode it is made in)
        torch = _torch()
        with torch.inference_mode(False):
            proto = _plain(torch.empty(0, dtype=torch.uint8 if dtype == "bytes" else _torch_dtype(dtype), device=like.device))
        proto.data_ptr()
        _empty[key] = proto
    value = proto.new_empty(shape)
    return value if type(value) is _Tensor else _plain(value)


def _like(value, dtype):
    """New memory of a tensor's kind and shape.  (For a plain tensor in half the time of ``_new``.)"""
    out = _torch().empty_like(value)
    return out if type(out) is _Tensor else _new(value, dtype, value.shape)


def _two(like, count):
    """Twice ``count`` new values of a float32 tensor's kind."""
    one, two = like.new_empty(count), like.new_empty(count)
    return (one, two) if type(one) is _Tensor else (_new(like, "f32", count), _new(like, "f32", count))


def _plain(value):
    if type(value) is not _Tensor:
        raise ValueError(f"the operators allocate memory of their own, not {type(value).__name__}s")
    return value


class Float8Tensor:
    """A float matrix ``[rows][channels]`` in 8 bits: codes in e4m3 or e5m2 and a power of two for every 128 consecutive channels of a
    row (of a weight: 128 x 128 elements), the least that brings the block's largest finite magnitude to the format's largest code.
    NaN stays NaN; an infinity becomes NaN in e4m3 and stays one in e5m2.  Made by ``float8_encode`` and by the operators; takes about
    ``rows * channels`` bytes (``nbytes``)."""

    def __init__(self, rows: int, channels: int, format: str, memory):
        """``memory``: contiguous uint8 CUDA tensor with the codes, then the exponents, 16-byte aligned (``lf_float8_matrix``)."""
        self.rows, self.channels, self.format, self.memory = rows, channels, _format(format), memory
        self._codes, exponents = _sizes(rows, channels)
        if memory.element_size() != 1 or not memory.is_cuda or not memory.is_contiguous():
            raise ValueError("memory must be a contiguous uint8 CUDA tensor")
        if memory.numel() != self._codes + exponents:
            raise RangeError(f"memory has {memory.numel()} values; expected {self._codes + exponents}")
        if type(memory) is not _Tensor:
            _has_memory("memory", memory)
        base = memory.data_ptr()
        self.fields = (rows, channels, _FORMAT[format], base, base + self._codes)

    @classmethod
    def empty(cls, rows, channels, format, like):
        codes, exponents = _sizes(rows, channels)
        return cls(rows, channels, format, _new(like, "bytes", codes + exponents))

    @property
    def nbytes(self):
        return self.memory.numel()

    @property
    def codes(self):
        """``[rows][channels rounded up to 16]`` bytes."""
        return self.memory[:self._codes].view(self.rows, -1)

    @property
    def exponents(self):
        """``[ceil(channels / 512)][ceil(rows / 128)][row % 32][row % 128 / 32][block % 4]`` bytes, 127 more than the powers."""
        return self.memory[self._codes:].view(-1, (self.rows + 127) // 128, 32, 4, 4)


def _matrix(device, name, value, rows, channels):
    if not isinstance(value, Float8Tensor):
        raise ValueError(f"{name} must be a Float8Tensor")
    if value.memory.get_device() != device.ordinal:
        raise ValueError(f"{name} is on {value.memory.device}, the device's GPU is cuda:{device.ordinal}")
    if (value.rows, value.channels) != (rows, channels):
        raise RangeError(f"{name} is {value.rows} x {value.channels}; expected {rows} x {channels}")
    return value


def _encode(device, source, dtype, out, block_rows=1, transposed=None, weights=None):
    desc = _ENCODE.pack(*out.fields, *(transposed.fields if transposed is not None else _NO_MATRIX), _DTYPE[dtype], block_rows, source.data_ptr())
    _call(device, device.lib.lf_float8_encode, desc, (source, out, transposed), weights=weights)


def float8_encode(device, activations, rows, channels, options=None):
    """The 8-bit form of ``activations`` ``[rows][channels]`` (float32 or bfloat16).  ``options``: format "e4m3" (default) or "e5m2"
    (more range, less precision: gradients)."""
    dev = _device(device)
    shape = {"rows": rows, "channels": channels}
    rows, channels = _size(shape, "rows"), _size(shape, "channels")
    format = _format((options or _NO_OPTIONS).get("format", "e4m3"))
    dtype = _tensor(dev, "activations", activations, rows * channels)
    out = Float8Tensor.empty(rows, channels, format, activations)
    _encode(dev, activations, dtype, out)
    return out


def float8_decode(device, encoded, options=None, out=None):
    """The values of a ``Float8Tensor`` as a tensor ``[rows][channels]``.  ``options``: output "bf16" (default) or "f32"; both hold them
    exactly (bf16 with its least step of 2^-133: blocks below about 2^-101 are rounded to it)."""
    dev = _device(device)
    if not isinstance(encoded, Float8Tensor):
        raise ValueError("encoded must be a Float8Tensor")
    _matrix(dev, "encoded", encoded, encoded.rows, encoded.channels)
    dtype, fresh = _output(options, "bf16"), out is None
    if fresh:
        out = _new(encoded.memory, dtype, (encoded.rows, encoded.channels))
    else:
        _tensor(dev, "out", out, encoded.rows * encoded.channels, dtype)
    _call(dev, dev.lib.lf_float8_decode, _DECODE.pack(*encoded.fields, _DTYPE[dtype], 0, out.data_ptr()), (encoded, out), fresh=fresh)
    return out


def _output(options, default):
    value = (options or _NO_OPTIONS).get("output") or default
    if value not in _DTYPE:
        raise ValueError(f'output must be "f32" or "bf16"; received {value!r}')
    return value


class LayerNormGpu:
    """LayerNorm over the channels of each row (at most 8192), and its gradients.  Statistics and sums are float32."""

    def __init__(self, device: Device | None = None):
        self.device = _device(device)

    def run(self, input, options=None, out=None):
        """``input``: rows, channels, activations ``[rows][channels]`` (float32 or bfloat16, as is the output), scale and offset
        ``[channels]`` (float32), epsilon (default 1e-5).  ``options``: statistics - also return ``mean`` and ``inverseDeviation``
        ``[rows]`` for ``backward``; checkpoint "e4m3" | "e5m2" - those and the input's 8-bit form as ``checkpoint``; encode "e4m3" |
        "e5m2" - the output is a ``Float8Tensor``, the operand of a ``Float8LinearGpu``; variance "two-pass" | "fast" (two passes
        either way).  ``out`` may be the activations; it may not overlap them otherwise."""
        dev, opts = self.device, options or _NO_OPTIONS
        rows, c = _size(input, "rows"), _size(input, "channels")
        x, scale, offset = input["activations"], input["scale"], input["offset"]
        epsilon = input.get("epsilon")
        epsilon = 1e-5 if epsilon is None else epsilon
        if not 0 < epsilon <= _LARGEST:
            raise RangeError(f"epsilon must be finite and positive; received {epsilon}")
        variance = _variance(opts, "two-pass") if opts else nat.VARIANCE_TWO_PASS
        kept, encode = opts.get("checkpoint"), opts.get("encode")
        kept = None if kept is None else _format(kept, "checkpoint")
        encode = None if encode is None else _format(encode, "encode")
        dtype = _tensor(dev, "activations", x, rows * c)
        _tensor(dev, "scale", scale, c, "f32")
        _tensor(dev, "offset", offset, c, "f32")
        if encode and out is not None:
            raise ValueError("an encoded output is a new Float8Tensor; out is for the other kind")
        given = out is not None
        if given:
            _tensor(dev, "out", out, rows * c, dtype)
        elif not encode:
            out = _like(x, dtype)
        checkpoint = Float8Tensor.empty(rows, c, kept, x) if kept else None
        encoded = Float8Tensor.empty(rows, c, encode, x) if encode else None
        mean = inverse = None
        statistics = kept or opts.get("statistics")
        if statistics:
            mean, inverse = _two(scale, rows)
        desc = _LAYER_NORM.pack(rows, c, variance, _DTYPE[dtype], epsilon, x.data_ptr(), scale.data_ptr(), offset.data_ptr(),
                                out.data_ptr() if out is not None else 0, 0 if mean is None else mean.data_ptr(), 0 if mean is None else inverse.data_ptr(),
                                *(checkpoint.fields if kept else _NO_MATRIX), *(encoded.fields if encode else _NO_MATRIX))
        result = _call(dev, dev.lib.lf_layer_norm_run, desc, (x, scale, offset, out, mean, inverse, checkpoint, encoded), encoded if encode else out, not given or bool(statistics))
        if mean is not None:
            result["mean"], result["inverseDeviation"] = mean, inverse
        if kept:
            result["checkpoint"] = checkpoint
        return result

    def backward(self, input, options=None, out=None):
        """``input``: rows, channels, gradient (of the output, ``[rows][channels]``), activations (the forward pass' input: a tensor of
        the gradient's type, or its checkpoint), mean, inverseDeviation, scale.  Returns the gradients of ``activations`` (of the
        gradient's type; ``out`` may be the gradient or the activations, and may not overlap them otherwise), ``scale`` and ``offset`` (float32).  The sums over the rows have a
        fixed order: the same call gives the same bits."""
        dev = self.device
        rows, c = _size(input, "rows"), _size(input, "channels")
        dy, x, scale, mean, inverse = input["gradient"], input["activations"], input["scale"], input["mean"], input["inverseDeviation"]
        dtype = _tensor(dev, "gradient", dy, rows * c)
        encoded = isinstance(x, Float8Tensor)
        if encoded:
            _matrix(dev, "activations", x, rows, c)
        else:
            _tensor(dev, "activations", x, rows * c, dtype)
        _tensor(dev, "mean", mean, rows, "f32")
        _tensor(dev, "inverseDeviation", inverse, rows, "f32")
        _tensor(dev, "scale", scale, c, "f32")
        if out is not None:
            _tensor(dev, "out", out, rows * c, dtype)
        else:
            out = _like(dy, dtype)
        nbytes = dev.lib.lf_layer_norm_backward_workspace(dev.handle, rows, c)
        dscale, doffset = _two(scale, c)
        workspace = _new(scale, "bytes", nbytes) if nbytes else None
        desc = _LAYER_NORM_BACKWARD.pack(rows, c, _DTYPE[dtype], dy.data_ptr(), 0 if encoded else x.data_ptr(), *(x.fields if encoded else _NO_MATRIX),
                                         mean.data_ptr(), inverse.data_ptr(), scale.data_ptr(), out.data_ptr(), dscale.data_ptr(), doffset.data_ptr(), workspace.data_ptr() if nbytes else 0, nbytes)
        result = _call(dev, dev.lib.lf_layer_norm_backward_run, desc, (dy, x, mean, inverse, scale, out, dscale, doffset, workspace), out)
        result["activations"] = result.pop("output")
        result["scale"], result["offset"] = dscale, doffset
        return result


class Float8LinearWeights:
    """A projection's weight ``[outChannels][channels]`` on the device in e4m3, one power of two for every 128 x 128 elements, in both
    orientations (the transposed one multiplies gradients), and its bias.  ``update`` encodes new values into the same memory, as
    a training step does; calls enqueued before it, on this device or another of the same GPU, have read the old ones.  Calls of another device wait for the
    weights; one that is captured cannot, and takes them as the first call after an update has found them.  Replays are ordered with updates by
    who replays."""

    _readers = None      # other devices of the GPU that have waited for the weights since the last update, and may still be reading
    _origin = None       # torch's current stream when the memory was allocated
    _elsewhere = None    # devices with calls on other streams, made while those were torch's current ones

    def __init__(self, device: Device, weight, bias=None):
        self.device = device
        shape = tuple(getattr(weight, "shape", ()))
        if len(shape) != 2:
            raise RangeError(f"weight must be [outChannels][channels]; received shape {shape}")
        self.out_channels, self.channels = int(shape[0]), int(shape[1])
        _positive("outChannels", self.out_channels)
        _positive("channels", self.channels)
        weight = self._on_device(weight)
        _tensor(device, "weight", weight, self.out_channels * self.channels)
        self.bias, self._origin = None, _torch_stream(device.ordinal)
        self.forward = Float8Tensor.empty(self.out_channels, self.channels, "e4m3", weight)
        self.transposed = Float8Tensor.empty(self.channels, self.out_channels, "e4m3", weight)
        self.update(weight, bias)

    def _read_on(self, device):
        if self._elsewhere is None:
            self._elsewhere = weakref.WeakSet()
        self._elsewhere.add(device)

    def __del__(self):
        """The memory goes back to the stream that it came from, which knows nothing of calls on others: their devices keep it until they are through.
        (What a graph reads, its caller keeps.)"""
        if self._elsewhere and not sys.is_finalizing() and not _capturing():
            for device in self._elsewhere:
                if device._finalizer.alive:
                    device.hold((self.forward, self.transposed))

    def _on_device(self, value):
        if value is None or getattr(value, "is_cuda", False):
            return value
        import torch
        host = value.decode() if isinstance(value, EncodedTensor) else np.ascontiguousarray(np.asarray(value, np.float32))
        return torch.as_tensor(host).to(f"cuda:{self.device.ordinal}")

    def update(self, weight, bias=_AS_IT_WAS):
        """A new weight (float32 or bfloat16 CUDA tensor, or host array) and, if given, a new bias (float32, or None).  The bias tensor is
        not copied: calls read what it holds."""
        if not self.device._finalizer.alive:
            raise ValueError("the weights' device is closed: they can be read, by other devices, and not updated")
        weight, bias = self._on_device(weight), self.bias if bias is _AS_IT_WAS else self._on_device(bias)
        if weight.shape != (self.out_channels, self.channels):
            raise RangeError(f"weight is {tuple(weight.shape)}; expected {(self.out_channels, self.channels)}")
        dtype = _tensor(self.device, "weight", weight, self.out_channels * self.channels)
        if bias is not None:
            _tensor(self.device, "bias", bias, self.out_channels, "f32")
        self.bias = bias
        for reader in self._readers or ():
            if reader._finalizer.alive:      # (a closed device has finished)
                self.device.check(self.device.lib.lf_context_await(self.device.handle, reader.stream))
        self._readers = None
        _encode(self.device, weight, dtype, self.forward, 128, self.transposed, self)


def prepare_float8_linear_weights(device, weight, bias=None):
    """``Float8LinearWeights`` of a ``[outChannels][channels]`` weight: a CUDA tensor, a host array or an ``EncodedTensor`` of a bundle."""
    return Float8LinearWeights(_device(device), weight, bias)


class Float8LinearGpu:
    """The projection ``y = x . weight^T + bias`` on 8-bit operands with float32 sums, and its gradients.  The sums are the tensor core's, which
    truncate: a product's error grows with its channels (2e-7 of it at 4096, 1e-6 at 16384, 5e-5 at 262144).

    ``run`` and ``input_gradient`` encode a float32 or bfloat16 operand in the call (``options``: format "e4m3" (default) | "e5m2") or take
    a ``Float8Tensor``; with the option checkpoint the encoded operand is returned as ``checkpoint``.  Option output "f32" | "bf16":
    the result's type, by default the operand's (bf16 for a ``Float8Tensor``).  ``out`` may not overlap what the call reads."""

    def __init__(self, device: Device | None = None):
        self.device = _device(device)

    def _product(self, name, value, rows, channels, prepared, weights, bias, options, out):
        dev, opts = self.device, options or _NO_OPTIONS
        keep, source, operand, workspace, nbytes = bool(opts.get("checkpoint")), None, None, None, 0
        format = _format(opts.get("format", "e4m3"))
        if isinstance(value, Float8Tensor):
            operand, dtype = _matrix(dev, name, value, rows, channels), _output(opts, "bf16")
        else:
            source = _tensor(dev, name, value, rows * channels)
            dtype = _output(opts, source)
            if keep:
                operand = Float8Tensor.empty(rows, channels, format, value)
            else:
                nbytes = dev.lib.lf_float8_linear_workspace(rows, channels)
                workspace = _new(value, "bytes", nbytes) if nbytes else None
        fresh = out is None or keep or nbytes > 0
        if out is not None:
            _tensor(dev, "out", out, rows * weights.rows, dtype)
        else:
            out = _new(weights.memory, dtype, (rows, weights.rows))
        desc = _LINEAR.pack(*(operand.fields if operand is not None else (rows, channels, _FORMAT[format], 0, 0)), *weights.fields,
                            bias.data_ptr() if bias is not None else 0, _DTYPE[dtype], _DTYPE[source or "f32"], value.data_ptr() if source else 0,
                            out.data_ptr(), workspace.data_ptr() if nbytes else 0, nbytes)
        result = _call(dev, dev.lib.lf_float8_linear_run, desc, (value, operand, weights, bias, workspace, out), out, fresh, prepared)
        if keep:
            result["checkpoint"] = operand
        return result

    def _weights(self, input):
        rows, channels, n = _size(input, "rows"), _size(input, "channels"), _size(input, "outChannels")
        weights = input["weights"]
        if not isinstance(weights, Float8LinearWeights):
            raise ValueError("weights must come from prepare_float8_linear_weights")
        if weights.device is not self.device:
            if weights.device.ordinal != self.device.ordinal:
                raise ValueError(f"weights are on cuda:{weights.device.ordinal}, the device's GPU is cuda:{self.device.ordinal}")
            if weights._readers is None:
                weights._readers = weakref.WeakSet()
            # (encoded on its stream, by a replayed graph perhaps; a captured call cannot wait and need not where one before it has)
            if weights.device._finalizer.alive and not (self.device in weights._readers and _capturing()):
                self.device.check(self.device.lib.lf_context_await(self.device.handle, weights.device.stream))
            weights._readers.add(self.device)
        if (weights.out_channels, weights.channels) != (n, channels):
            raise RangeError(f"weights are {weights.out_channels} x {weights.channels}; expected {n} x {channels}")
        return rows, channels, n, weights

    def run(self, input, options=None, out=None):
        """``input``: rows, channels, outChannels, activations ``[rows][channels]``, weights -> ``output`` ``[rows][outChannels]``."""
        rows, channels, _, weights = self._weights(input)
        return self._product("activations", input["activations"], rows, channels, weights, weights.forward, weights.bias, options, out)

    def input_gradient(self, input, options=None, out=None):
        """``input``: rows, channels, outChannels, gradient ``[rows][outChannels]``, weights -> ``output`` ``[rows][channels]``, the
        gradient of the activations."""
        rows, _, n, weights = self._weights(input)
        return self._product("gradient", input["gradient"], rows, n, weights, weights.transposed, None, options, out)

    def weight_gradient(self, input, options=None):
        """``input``: rows, channels, outChannels, gradient ``[rows][outChannels]`` (bfloat16 or a ``Float8Tensor``; a float32 gradient is
        encoded first, ``float8_encode``), activations (the ``Float8Tensor`` that the forward pass multiplied with) -> ``weight``
        ``[outChannels][channels]`` and ``bias`` ``[outChannels]``, float32, the same bits at every call.  Both are sums over the gradient as given: of an encoded one the
        bias' gradient adds up the 8-bit values, not those that they were made from."""
        dev = self.device
        rows, channels, n = _size(input, "rows"), _size(input, "channels"), _size(input, "outChannels")
        if max(channels, n) > _MOST_GRADIENT:
            raise NotImplementedError(f"the weight's gradient of {n} x {channels} channels: at most {_MOST_GRADIENT} of either")
        dy, x = input["gradient"], _matrix(dev, "activations", input["activations"], rows, channels)
        encoded = isinstance(dy, Float8Tensor)
        if encoded:
            _matrix(dev, "gradient", dy, rows, n)
        else:
            _tensor(dev, "gradient", dy, rows * n, "bf16")
        nbytes = dev.lib.lf_float8_weight_gradient_workspace(dev.handle, rows, channels, n)
        weight = _new(x.memory, "f32", (n, channels))
        bias, workspace = weight.new_empty(n), _new(weight, "bytes", nbytes) if nbytes else None
        desc = _WEIGHT_GRADIENT.pack(*x.fields, 0 if encoded else dy.data_ptr(), *(dy.fields if encoded else _NO_MATRIX), n, 0, weight.data_ptr(), bias.data_ptr(),
                                     workspace.data_ptr() if nbytes else 0, nbytes)
        result = _call(dev, dev.lib.lf_float8_weight_gradient_run, desc, (dy, x, weight, bias, workspace), weight)
        result["weight"] = result.pop("output")
        result["bias"] = bias
        return result
