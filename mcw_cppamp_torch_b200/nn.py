"""The `nn` modules on the hot path, mirroring the reference's Lua classes over the C ABI.

Each class keeps the field names the reference's C operators read off the Lua module table
(`weight`, `bias`, `gradWeight`, `gradBias`, `finput`, `fgradInput`, `output`, `gradInput`,
`indices`, `kW`, `kH`, `dW`, `dH`, `padding`, `threshold`, `val`) and the `nn.Module` protocol of
mcw_nn/Module.lua:20-82 (forward / backward / updateOutput / updateGradInput / accGradParameters /
zeroGradParameters / updateParameters / parameters / getParameters).  Modules are built with host
(numpy) parameters, like the reference builds them with FloatTensors, and `:gpu()` moves them.
There is no CPU compute path: calling forward before `:gpu()` raises."""
import ctypes as C
import math

import numpy as np

from ._lib import lib
from .tensor import GPUTensor, gpu, _long_storage


class _NumpyRng:
    """Default host RNG for `reset()`; tests pass the TH-compatible generator instead."""

    def __init__(self, seed=0):
        self._g = np.random.default_rng(seed)

    def uniform(self, shape, a, b):
        return self._g.uniform(a, b, size=shape).astype(np.float32)


_default_rng = _NumpyRng()


def _need_gpu(t, what):
    if not isinstance(t, GPUTensor):
        raise TypeError("%s: torch.GPUTensor expected (this build has no CPU compute path; call :gpu())" % what)
    return t


class Module:
    """mcw_nn/Module.lua"""

    def __init__(self):
        self.output = GPUTensor()
        self.gradInput = GPUTensor()

    # -- protocol --
    def parameters(self):
        w, g = [], []
        if getattr(self, "weight", None) is not None:
            w += [self.weight]; g += [self.gradWeight]
        if getattr(self, "bias", None) is not None:
            w += [self.bias]; g += [self.gradBias]
        return (w, g) if w else None

    def updateOutput(self, input):
        return self.output

    def updateGradInput(self, input, gradOutput):
        return self.gradInput

    def accGradParameters(self, input, gradOutput, scale=1.0):
        pass

    def forward(self, input):
        return self.updateOutput(input)

    def backward(self, input, gradOutput, scale=1.0):
        self.updateGradInput(input, gradOutput)
        self.accGradParameters(input, gradOutput, scale)
        return self.gradInput

    def zeroGradParameters(self):
        p = self.parameters()
        if p:
            for g in p[1]:
                g.zero()

    def updateParameters(self, learningRate):
        p = self.parameters()
        if p:
            for w, g in zip(*p):
                w.add(-learningRate, g)

    def gpu(self):
        """Module:type('torch.GPUTensor'): converts every host tensor field (mcw_nn/Module.lua:116-148)."""
        for k, v in list(self.__dict__.items()):
            if isinstance(v, np.ndarray):
                setattr(self, k, gpu(v))
        return self

    def training(self):
        """mcw_nn/Dropout.lua's `train` field for every module: forward passes keep what a backward pass reads."""
        return self._set_train(True)

    def evaluate(self):
        return self._set_train(False)

    def _set_train(self, on):
        for m in self.modules_list():
            m.train = on
        return self

    def modules_list(self):
        return [self]

    def clone(self):
        """mcw_nn/Module.lua:104-114: the module written into a memory file and read back -- every GPU tensor
        goes through the library's storage / tensor records, tensors that share a storage still share one."""
        import io
        import pickle
        buf = io.BytesIO()
        pickle.dump(self, buf, protocol=4)
        buf.seek(0)
        return pickle.load(buf)

    def getParameters(self, flat=None):
        """Flattens all parameters (and gradients) into one storage each and re-points the modules'
        tensors at views of it (mcw_nn/Module.lua:169-252).  `flat` may carry two caller-owned
        device buffers `(w_ptr, g_ptr, n)` to flatten into (e.g. memory shared with a collective)."""
        L = lib()
        ws, gs = [], []
        for m in self.modules_list():
            p = m.parameters()
            if p:
                ws += p[0]; gs += p[1]
        n = sum(t.nElement() for t in ws)
        if flat is None:
            fw, fg = GPUTensor(n), GPUTensor(n)
        else:
            wptr, gptr, cap = flat
            assert cap >= n
            sw = L.THGPUStorage_newWithData(C.c_void_p(wptr), n)
            sg = L.THGPUStorage_newWithData(C.c_void_p(gptr), n)
            fw = GPUTensor(_ptr=L.THGPUTensor_newWithStorage1d(sw, 0, n, 1))
            fg = GPUTensor(_ptr=L.THGPUTensor_newWithStorage1d(sg, 0, n, 1))
            L.THGPUStorage_free(sw); L.THGPUStorage_free(sg)
        off = 0
        for t, g in zip(ws, gs):
            k = t.nElement()
            for flat_t, part in ((fw, t), (fg, g)):
                dst = flat_t.narrow(1, off + 1, k)
                dst.copy(part.contiguous().view(k))
                size = _long_storage(list(part.size()))
                L.THGPUTensor_setStorage(part._p, flat_t._p.contents.storage, off, C.byref(size), None)
            off += k
        return fw, fg


class Sequential(Module):
    """mcw_nn/Sequential.lua"""

    def __init__(self):
        super().__init__()
        self.modules = []

    def add(self, m):
        self.modules.append(m)
        return self

    def modules_list(self):
        out = []
        for m in self.modules:
            out += m.modules_list()
        return out

    def parameters(self):
        return None

    def gpu(self):
        for m in self.modules:
            m.gpu()
        return self

    def updateOutput(self, input):
        cur, ms, i = input, self.modules, 0
        while i < len(ms):
            if i + 1 < len(ms) and _threshold_pool(ms[i], ms[i + 1], "forward"):
                cur = _threshold_pool_forward(ms[i], ms[i + 1], cur)
                i += 2
            else:
                cur = ms[i].updateOutput(cur)
                i += 1
        self.output = cur
        return cur

    def _back(self, input, gradOutput, step):
        """`step(module, its input, its gradOutput)` from the last module to the first"""
        cur, ms = gradOutput, self.modules
        i = len(ms) - 1
        if i < 0:
            raise IndexError("Sequential without modules")
        while i >= 0:
            if i > 0 and _threshold_pool(ms[i - 1], ms[i], "backward"):
                cur = _threshold_pool_backward(ms[i - 1], ms[i], ms[i - 2].output if i > 1 else input, cur)
                i -= 2
            else:
                cur = step(ms[i], ms[i - 1].output if i > 0 else input, cur)
                i -= 1
        self.gradInput = cur
        return cur

    def updateGradInput(self, input, gradOutput):
        return self._back(input, gradOutput, lambda m, x, g: m.updateGradInput(x, g))

    def accGradParameters(self, input, gradOutput, scale=1.0):
        cur = gradOutput
        for i in range(len(self.modules) - 1, 0, -1):
            prev = self.modules[i - 1].output
            self.modules[i].accGradParameters(prev, cur, scale)
            cur = self.modules[i].gradInput
        self.modules[0].accGradParameters(input, cur, scale)

    def backward(self, input, gradOutput, scale=1.0):
        # mcw_nn/Sequential.lua backward: each module's backward in reverse order
        return self._back(input, gradOutput, lambda m, x, g: m.backward(x, g, scale))

    def zeroGradParameters(self):
        for m in self.modules:
            m.zeroGradParameters()

    def updateParameters(self, lr):
        for m in self.modules:
            m.updateParameters(lr)


class SpatialConvolutionMM(Module):
    """mcw_nn/SpatialConvolutionMM.lua over gpunn SpatialConvolutionMM_* (reference:
    gputorch/lib/THC/gpunn-impl/SpatialConvolutionMM.cpp:110-429)."""

    def __init__(self, nInputPlane, nOutputPlane, kW, kH, dW=1, dH=1, padding=0, rng=None):
        super().__init__()
        self.nInputPlane, self.nOutputPlane = nInputPlane, nOutputPlane
        self.kW, self.kH, self.dW, self.dH, self.padding = kW, kH, dW, dH, padding
        self.weight = np.empty((nOutputPlane, nInputPlane * kH * kW), np.float32)
        self.bias = np.empty((nOutputPlane,), np.float32)
        self.gradWeight = np.zeros_like(self.weight)
        self.gradBias = np.zeros_like(self.bias)
        self.finput = GPUTensor()
        self.fgradInput = GPUTensor()
        self.reset(rng=rng)

    def reset(self, stdv=None, rng=None):
        """uniform(-stdv, stdv), weight first then bias (mcw_nn/SpatialConvolutionMM.lua:29-46)."""
        rng = rng or _default_rng
        stdv = stdv * math.sqrt(3) if stdv else 1.0 / math.sqrt(self.kW * self.kH * self.nInputPlane)
        w = rng.uniform(tuple(self.weight.shape) if isinstance(self.weight, np.ndarray) else self.weight.size(), -stdv, stdv)
        b = rng.uniform((self.nOutputPlane,), -stdv, stdv)
        if isinstance(self.weight, np.ndarray):
            self.weight, self.bias = w, b
        else:
            self.weight.copy(w); self.bias.copy(b)

    def updateOutput(self, input):
        _need_gpu(input, "SpatialConvolutionMM"); _need_gpu(self.weight, "SpatialConvolutionMM.weight")
        lib().THGPUNN_SpatialConvolutionMM_updateOutput(input._p, self.output._p, self.weight._p, self.bias._p,
                                                        self.finput._p, self.fgradInput._p, self.kW, self.kH,
                                                        self.dW, self.dH, self.padding)
        return self.output

    def updateGradInput(self, input, gradOutput):
        if self.gradInput is None:
            return None
        lib().THGPUNN_SpatialConvolutionMM_updateGradInput(input._p, gradOutput._p, self.gradInput._p, self.weight._p,
                                                           self.finput._p, self.fgradInput._p, self.kW, self.kH,
                                                           self.dW, self.dH, self.padding)
        return self.gradInput

    def accGradParameters(self, input, gradOutput, scale=1.0):
        lib().THGPUNN_SpatialConvolutionMM_accGradParameters(input._p, gradOutput._p, self.gradWeight._p,
                                                             self.gradBias._p, self.finput._p, self.fgradInput._p,
                                                             self.kW, self.kH, self.dW, self.dH, self.padding, scale)


    def backward(self, input, gradOutput, scale=1.0):
        """updateGradInput + accGradParameters (mcw_nn/Module.lua backward) in one library call that
        transposes gradOutput once."""
        gi = self.gradInput._p if self.gradInput is not None else None
        lib().THGPUNN_SpatialConvolutionMM_backward(input._p, gradOutput._p, gi, self.weight._p, self.gradWeight._p,
                                                    self.gradBias._p, self.finput._p, self.fgradInput._p,
                                                    self.kW, self.kH, self.dW, self.dH, self.padding, scale)
        return self.gradInput


class SpatialMaxPooling(Module):
    """mcw_nn/SpatialMaxPooling.lua over gpunn SpatialMaxPooling_*."""

    def __init__(self, kW, kH, dW=None, dH=None):
        super().__init__()
        self.kW, self.kH = kW, kH
        self.dW, self.dH = dW or kW, dH or kH
        self.indices = GPUTensor()

    def updateOutput(self, input):
        _need_gpu(input, "SpatialMaxPooling")
        lib().THGPUNN_SpatialMaxPooling_updateOutput(input._p, self.output._p, self.indices._p, self.kW, self.kH,
                                                     self.dW, self.dH)
        return self.output

    def updateGradInput(self, input, gradOutput):
        lib().THGPUNN_SpatialMaxPooling_updateGradInput(input._p, gradOutput._p, self.gradInput._p, self.indices._p,
                                                        self.kW, self.kH, self.dW, self.dH)
        return self.gradInput


class Threshold(Module):
    """mcw_nn/Threshold.lua"""

    def __init__(self, th=1e-6, v=0.0):
        super().__init__()
        self.threshold, self.val = th, v

    def updateOutput(self, input):
        _need_gpu(input, "Threshold")
        lib().THGPUNN_Threshold_updateOutput(input._p, self.output._p, self.threshold, self.val)
        return self.output

    def updateGradInput(self, input, gradOutput):
        lib().THGPUNN_Threshold_updateGradInput(input._p, gradOutput._p, self.gradInput._p, self.threshold)
        return self.gradInput


class ReLU(Threshold):
    """mcw_nn/ReLU.lua:3-5: Threshold(0, 0)"""

    def __init__(self):
        super().__init__(0.0, 0.0)


# A Threshold and the SpatialMaxPooling behind it in one library call, which leaves in both what their own calls leave.  Only for modules
# of these very classes that nothing overrides.
_FORWARD, _BACKWARD = ("updateOutput",), ("backward", "updateGradInput", "accGradParameters")
_STOCK = {c: {n: getattr(c, n) for n in _FORWARD + _BACKWARD} for c in (Threshold, ReLU, SpatialMaxPooling)}


def _stock(m, names):
    c = type(m)
    return all(getattr(c, n) is _STOCK[c][n] and n not in m.__dict__ for n in names)


def _threshold_pool(a, b, way):
    if type(b) is not SpatialMaxPooling or type(a) not in (Threshold, ReLU):
        return False
    names = _FORWARD if way == "forward" else _BACKWARD
    return _stock(a, names) and _stock(b, names)


def _threshold_pool_forward(a, b, input):
    _need_gpu(input, "Threshold")
    lib().THGPUNN_Threshold_SpatialMaxPooling_updateOutput(input._p, a.output._p, b.output._p, b.indices._p, a.threshold, a.val,
                                                           b.kW, b.kH, b.dW, b.dH)
    return b.output


def _threshold_pool_backward(a, b, input, gradOutput):
    lib().THGPUNN_Threshold_SpatialMaxPooling_updateGradInput(input._p, a.output._p, gradOutput._p, b.gradInput._p, a.gradInput._p, b.indices._p,
                                                              a.threshold, b.kW, b.kH, b.dW, b.dH)
    return a.gradInput


class View(Module):
    """Reshape of a contiguous batch, e.g. [N,256,6,6] -> [N,9216] (mcw_nn/Reshape.lua / View)."""

    def __init__(self, *sizes):
        super().__init__()
        self.sizes = sizes

    def updateOutput(self, input):
        n = input.size(1)
        self.output = input.contiguous().view(n, *self.sizes)
        return self.output

    def updateGradInput(self, input, gradOutput):
        self.gradInput = gradOutput.contiguous().view(*input.size())
        return self.gradInput


class Linear(Module):
    """mcw_nn/Linear.lua:33-94, batch mode: addmm for the products, the bias added in the forward product's epilogue."""

    def __init__(self, inputSize, outputSize, rng=None):
        super().__init__()
        self.weight = np.empty((outputSize, inputSize), np.float32)
        self.bias = np.empty((outputSize,), np.float32)
        self.gradWeight = np.zeros((outputSize, inputSize), np.float32)
        self.gradBias = np.zeros((outputSize,), np.float32)
        self._ones = None
        self.reset(rng=rng)

    def reset(self, stdv=None, rng=None):
        rng = rng or _default_rng
        shape = tuple(self.weight.shape) if isinstance(self.weight, np.ndarray) else self.weight.size()
        stdv = stdv * math.sqrt(3) if stdv else 1.0 / math.sqrt(shape[1])
        w = rng.uniform(shape, -stdv, stdv)
        b = rng.uniform((shape[0],), -stdv, stdv)
        if isinstance(self.weight, np.ndarray):
            self.weight, self.bias = w, b
        else:
            self.weight.copy(w); self.bias.copy(b)

    def _ones_vec(self, n):
        if self._ones is None or self._ones.nElement() != n:
            self._ones = GPUTensor(n).fill(1)
        return self._ones

    def updateOutput(self, input):
        _need_gpu(input, "Linear"); _need_gpu(self.weight, "Linear.weight")
        assert input.dim() == 2, "batch (2-D) input expected"
        lib().THGPUNN_Linear_updateOutput(input._p, self.output._p, self.weight._p, self.bias._p)
        return self.output

    def updateGradInput(self, input, gradOutput):
        if self.gradInput is None:
            return None
        self.gradInput.resizeAs(input)
        self.gradInput.addmm(0, 1, gradOutput, self.weight)
        return self.gradInput

    def accGradParameters(self, input, gradOutput, scale=1.0):
        self.gradWeight.addmm(scale, gradOutput.t(), input)
        self.gradBias.addmv(scale, gradOutput.t(), self._ones_vec(input.size(1)))


ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}


def _activation(name):
    if name not in ACTIVATIONS:
        raise ValueError("activation %r: one of %s expected" % (name, ", ".join(ACTIVATIONS)))
    return ACTIVATIONS[name]


def _need_kept(m):
    if not m._kept:
        raise RuntimeError("%s: the last forward pass has kept nothing for a backward pass (it ran after evaluate())" % type(m).__name__)


class LayerNorm(Module):
    """Rows normalised to mean zero and variance one over the trailing `sizes`, times `weight` plus `bias` (one of each for every place
    in a row); with affine=False the normalised rows themselves.  An input may have neighbours among the sizes as one dimension, or one of
    them as several.  `mean` and `invStd` keep each row's statistics for the backward pass; after evaluate() they are left alone."""
    sizes = ()

    def __init__(self, *sizes, eps=1e-5, affine=True):
        super().__init__()
        self.size, self.eps, self.train, self._kept = math.prod(sizes), eps, True, True
        if not sizes or min(sizes) < 1:
            raise ValueError("LayerNorm: positive sizes expected")
        self.sizes = sizes
        self.mean, self.invStd = GPUTensor(), GPUTensor()
        self.weight = self.bias = self.gradWeight = self.gradBias = None
        if affine:
            self.weight, self.bias = np.ones(self.size, np.float32), np.zeros(self.size, np.float32)
            self.gradWeight, self.gradBias = np.zeros(self.size, np.float32), np.zeros(self.size, np.float32)

    def _affine(self):
        if self.weight is None:
            return None, None
        return _need_gpu(self.weight, "LayerNorm.weight")._p, self.bias._p

    def _ends(self, sizes):
        """How many values each of the last dimensions has with those behind it, up to a row's."""
        n, ends = 1, set()
        for k in reversed(sizes):
            if n >= self.size:
                break
            n *= k
            ends.add(n)
        return ends

    def updateOutput(self, input):
        _need_gpu(input, "LayerNorm")
        if len(self.sizes) > 1:
            mine, its = self._ends(self.sizes), self._ends(input.size())
            if not (mine <= its or its <= mine):
                raise ValueError("LayerNorm: trailing sizes %s expected, not those of %s" % (self.sizes, tuple(input.size())))
        w, b = self._affine()
        keep = (self.mean._p, self.invStd._p) if self.train else (None, None)
        lib().THGPUNN_LayerNorm_updateOutput(input._p, self.output._p, w, b, keep[0], keep[1], self.size, self.eps)
        self._kept = self.train
        return self.output

    def _back(self, input, gradOutput, gradInput, gradWeight, gradBias, scale):
        _need_kept(self)
        lib().THGPUNN_LayerNorm_backward(input._p, gradOutput._p, gradInput, self._affine()[0], gradWeight, gradBias, self.mean._p, self.invStd._p,
                                         self.size, scale)

    def updateGradInput(self, input, gradOutput):
        if self.gradInput is None:
            return None
        self._back(input, gradOutput, self.gradInput._p, None, None, 1.0)
        return self.gradInput

    def accGradParameters(self, input, gradOutput, scale=1.0):
        if self.weight is not None:
            self._back(input, gradOutput, None, self.gradWeight._p, self.gradBias._p, scale)

    def backward(self, input, gradOutput, scale=1.0):
        """updateGradInput + accGradParameters in one library call."""
        gi = self.gradInput._p if self.gradInput is not None else None
        gw, gb = (self.gradWeight._p, self.gradBias._p) if self.weight is not None else (None, None)
        self._back(input, gradOutput, gi, gw, gb, scale)
        return self.gradInput


class FusedLinear(Linear):
    """activation(input * weight^T + bias), or that plus a residual for the input [rows, residual], in one product whose epilogue does the
    rest.  activation: "none", "relu", "gelu" (of the normal distribution's integral) or "silu".  `preactivation` keeps the sum that the
    activation is taken of for the backward pass; after evaluate() forward passes leave it alone.
    With a residual gradInput is [the rows' gradient, gradOutput]: the second is the given tensor itself, which is not saved or cloned with the
    module."""

    def __init__(self, inputSize, outputSize, activation="none", rng=None):
        super().__init__(inputSize, outputSize, rng=rng)
        self.activation, self.train, self._kept = activation, True, True
        self._code = _activation(activation)
        self.preactivation, self.gradPreactivation = GPUTensor(), GPUTensor()

    def _split(self, input):
        if isinstance(input, (list, tuple)):
            rows, residual = input
            return _need_gpu(rows, type(self).__name__), _need_gpu(residual, type(self).__name__ + " residual")
        return _need_gpu(input, type(self).__name__), None

    def updateOutput(self, input):
        x, residual = self._split(input)
        _need_gpu(self.weight, "FusedLinear.weight")
        keep = self.preactivation._p if self.train and self._code else None
        lib().THGPUNN_FusedLinear_updateOutput(x._p, residual._p if residual is not None else None, self.output._p, keep, self.weight._p, self.bias._p,
                                               self._code)
        self._kept = self.train or not self._code
        return self.output

    def _back(self, input, gradOutput, gradInput, gradWeight, gradBias, scale):
        x, residual = self._split(input)
        _need_kept(self)
        lib().THGPUNN_FusedLinear_backward(x._p, gradOutput._p, gradInput, self.preactivation._p, self.gradPreactivation._p, self.weight._p, gradWeight,
                                           gradBias, self._code, scale)
        return residual

    def _grad_rows(self):
        """The rows' gradient in `gradInput`, which is a pair after a call with a residual."""
        return self.gradInput[0] if isinstance(self.gradInput, list) else self.gradInput

    def __getstate__(self):
        return dict(self.__dict__, gradInput=self._grad_rows())

    def updateGradInput(self, input, gradOutput):
        gi = self._grad_rows()
        if gi is None:
            return None
        residual = self._back(input, gradOutput, gi._p, None, None, 1.0)
        self.gradInput = gi if residual is None else [gi, gradOutput]
        return self.gradInput

    def accGradParameters(self, input, gradOutput, scale=1.0):
        self._back(input, gradOutput, None, self.gradWeight._p, self.gradBias._p, scale)

    def backward(self, input, gradOutput, scale=1.0):
        """updateGradInput + accGradParameters in one library call, which takes the activation's slope once."""
        gi = self._grad_rows()
        residual = self._back(input, gradOutput, gi._p if gi is not None else None, self.gradWeight._p, self.gradBias._p, scale)
        if gi is not None:
            self.gradInput = gi if residual is None else [gi, gradOutput]
        return self.gradInput


class GroupedLinear(Module):
    """activation(input * weight[e]^T + bias[e]) for the rows of group e: a layer of experts.  The input is [rows, counts], the rows sorted by
    group and `counts` a host sequence with the number of rows of each group (zeros among them): what Dispatch makes of rows and their experts'
    numbers, and Combine joins again.  weight is [groups, outputSize, inputSize], bias
    [groups, outputSize]; gradients of groups without rows stay as they are.  gradInput is [the rows' gradient, None].
    `activation`, `preactivation` and evaluate() as for FusedLinear.  In the "bf16" math mode the products stay FP32-accurate."""

    def __init__(self, groups, inputSize, outputSize, activation="none", rng=None):
        super().__init__()
        self.groups, self.activation, self.train, self._kept = groups, activation, True, True
        self._code = _activation(activation)
        self.weight = np.empty((groups, outputSize, inputSize), np.float32)
        self.bias = np.empty((groups, outputSize), np.float32)
        self.gradWeight = np.zeros((groups, outputSize, inputSize), np.float32)
        self.gradBias = np.zeros((groups, outputSize), np.float32)
        self.preactivation, self.gradPreactivation = GPUTensor(), GPUTensor()
        self.reset(rng=rng)

    def reset(self, stdv=None, rng=None):
        """Each group as Linear.reset draws a layer's."""
        rng = rng or _default_rng
        host = isinstance(self.weight, np.ndarray)
        shape = tuple(self.weight.shape) if host else self.weight.size()
        stdv = stdv * math.sqrt(3) if stdv else 1.0 / math.sqrt(shape[2])
        w, b = rng.uniform(shape, -stdv, stdv), rng.uniform(shape[:2], -stdv, stdv)
        if host:
            self.weight, self.bias = w, b
        else:
            self.weight.copy(w); self.bias.copy(b)

    def _split(self, input):
        x, counts = input
        if isinstance(counts, GPUTensor):
            raise TypeError("GroupedLinear: counts are a host sequence")
        counts = np.asarray(counts)
        if counts.shape != (self.groups,) or counts.dtype.kind not in "iu":
            raise ValueError("GroupedLinear: one whole number of rows for each of %d groups expected" % self.groups)
        return _need_gpu(x, "GroupedLinear"), np.ascontiguousarray(counts, np.int64)

    def updateOutput(self, input):
        x, counts = self._split(input)
        _need_gpu(self.weight, "GroupedLinear.weight")
        keep = self.preactivation._p if self.train and self._code else None
        lib().THGPUNN_GroupedLinear_updateOutput(x._p, counts, self.groups, self.output._p, keep, self.weight._p, self.bias._p, self._code)
        self._kept = self.train or not self._code
        return self.output

    def _back(self, input, gradOutput, gradInput, gradWeight, gradBias, scale):
        x, counts = self._split(input)
        _need_kept(self)
        lib().THGPUNN_GroupedLinear_backward(x._p, counts, self.groups, gradOutput._p, gradInput, self.preactivation._p, self.gradPreactivation._p,
                                             self.weight._p, gradWeight, gradBias, self._code, scale)

    def _grad_rows(self):
        return self.gradInput[0] if isinstance(self.gradInput, list) else self.gradInput

    def updateGradInput(self, input, gradOutput):
        gi = self._grad_rows()
        if gi is None:
            return None
        self._back(input, gradOutput, gi._p, None, None, 1.0)
        self.gradInput = [gi, None]
        return self.gradInput

    def accGradParameters(self, input, gradOutput, scale=1.0):
        self._back(input, gradOutput, None, self.gradWeight._p, self.gradBias._p, scale)

    def backward(self, input, gradOutput, scale=1.0):
        """updateGradInput + accGradParameters in one library call."""
        gi = self._grad_rows()
        self._back(input, gradOutput, gi._p if gi is not None else None, self.gradWeight._p, self.gradBias._p, scale)
        if gi is not None:
            self.gradInput = [gi, None]
        return self.gradInput


class Router(Module):
    """The k largest of each row's scores and softmax weights over them: output is [weights, experts], [rows, k] each, in descending order of the
    scores, equal ones by their place.  Experts are counted from 1.  A score of minus infinity closes its expert to the row; slots for which there is no open expert
    left, as in the rows of a padded batch, have the number 0 and the weight 0.  normalize: a row's weights sum to one, else they are those of the
    softmax over all its scores.  gradOutput is the weights' gradient, or [the weights' gradient, None]."""

    def __init__(self, k, normalize=True):
        super().__init__()
        if k < 1:
            raise ValueError("Router: at least one expert a row expected")
        self.k, self.normalize = k, normalize
        self.output = [GPUTensor(), GPUTensor()]

    def updateOutput(self, input):
        _need_gpu(input, "Router")
        lib().THGPUNN_Router_updateOutput(input._p, self.output[0]._p, self.output[1]._p, self.k, int(self.normalize))
        return self.output

    def updateGradInput(self, input, gradOutput):
        if self.gradInput is None:
            return None
        g = gradOutput[0] if isinstance(gradOutput, (list, tuple)) else gradOutput
        lib().THGPUNN_Router_updateGradInput(_need_gpu(input, "Router")._p, _need_gpu(g, "Router")._p, self.gradInput._p, self.output[0]._p, self.output[1]._p,
                                             int(self.normalize))
        return self.gradInput


class Dispatch(Module):
    """Rows sorted by the experts they go to: of the input [rows, experts], experts [rows, k] as Router leaves them (numbers from 1 to `groups`, 0: none),
    output is [a copy of a row for each of its experts, counts], sorted by expert, then by row, with the number of rows of each expert as a host array: GroupedLinear's
    input.  `positions` [rows, k] keeps the place of each copy, from 1 (0: none), for Combine and the backward pass.  A forward pass waits for the counts, so that
    it cannot be recorded.  gradOutput is [the copies' gradient, None] or that gradient itself; gradInput is [the rows' gradient, None]."""

    def __init__(self, groups):
        super().__init__()
        if groups < 1:
            raise ValueError("Dispatch: at least one group expected")
        self.groups = groups
        self.rows, self.positions, self.gradRows = GPUTensor(), GPUTensor(), GPUTensor()

    def updateOutput(self, input):
        x, experts = input
        counts = np.zeros(self.groups, np.int64)
        lib().THGPUNN_Dispatch_updateOutput(_need_gpu(x, "Dispatch")._p, _need_gpu(experts, "Dispatch experts")._p, self.rows._p, self.positions._p, counts, self.groups)
        self.output = [self.rows, counts]
        return self.output

    def updateGradInput(self, input, gradOutput):
        if self.gradInput is None:
            return None
        g = gradOutput[0] if isinstance(gradOutput, (list, tuple)) else gradOutput
        lib().THGPUNN_Dispatch_updateGradInput(_need_gpu(input[0], "Dispatch")._p, _need_gpu(g, "Dispatch")._p, self.gradRows._p, self.positions._p)
        self.gradInput = [self.gradRows, None]
        return self.gradInput


class Combine(Module):
    """The sum of each token's rows times their weights: of the input [rows, weights, positions] or [rows, weights, positions, residual], rows sorted as by
    Dispatch and weights and positions [tokens, k] (weights None: all one), plus the residual [tokens, size].  Slots whose position is 0 add nothing.
    A row is one slot's: the backward pass writes its gradient once.  `size` is needed where there may be no rows at all and no residual.
    gradInput is [the rows' gradient, the weights', None] or with a residual [the rows' gradient, the weights', None, gradOutput], the last the
    given tensor itself, which is not saved or cloned with the module.  Rows that no position names, as when some are set to 0 behind Dispatch, have zeros for their gradient."""

    def __init__(self, size=None):
        super().__init__()
        self.size = size
        self.gradRows, self.gradWeights = GPUTensor(), GPUTensor()

    def _split(self, input):
        rows, weights, positions, residual = input if len(input) == 4 else (*input, None)
        if weights is not None:
            _need_gpu(weights, "Combine weights")
        if residual is not None:
            _need_gpu(residual, "Combine residual")
        return _need_gpu(rows, "Combine"), weights, _need_gpu(positions, "Combine positions"), residual

    def updateOutput(self, input):
        rows, weights, positions, residual = self._split(input)
        size = self.size
        if size is None:
            sizes = rows.size() or (residual.size() if residual is not None else ())
            if len(sizes) != 2:
                if positions.dim():
                    raise ValueError("Combine: a matrix of rows expected, or the size of one in their place")
                sizes = (0, 1)                   # nothing to sum
            size = sizes[1]
        lib().THGPUNN_Combine_updateOutput(rows._p, weights._p if weights is not None else None, positions._p, residual._p if residual is not None else None,
                                           self.output._p, size)
        return self.output

    def updateGradInput(self, input, gradOutput):
        if self.gradInput is None:
            return None
        rows, weights, positions, residual = self._split(input)
        lib().THGPUNN_Combine_backward(rows._p, weights._p if weights is not None else None, positions._p, _need_gpu(gradOutput, "Combine")._p, self.gradRows._p,
                                       self.gradWeights._p if weights is not None else None)
        self.gradInput = [self.gradRows, self.gradWeights if weights is not None else None, None] + ([gradOutput] if residual is not None else [])
        return self.gradInput

    def __getstate__(self):
        return dict(self.__dict__, gradInput=self.gradInput[:3] if isinstance(self.gradInput, list) else self.gradInput)


class LogSoftMax(Module):
    """mcw_nn/LogSoftMax.lua"""

    def updateOutput(self, input):
        _need_gpu(input, "LogSoftMax")
        lib().THGPUNN_LogSoftMax_updateOutput(input._p, self.output._p)
        return self.output

    def updateGradInput(self, input, gradOutput):
        lib().THGPUNN_LogSoftMax_updateGradInput(input._p, gradOutput._p, self.gradInput._p, self.output._p)
        return self.gradInput


class SoftMax(Module):
    """mcw_nn/SoftMax.lua over gpunn SoftMax_* (gputorch/lib/THC/gpunn-impl/SoftMax.cpp)."""

    def updateOutput(self, input):
        _need_gpu(input, "SoftMax")
        lib().THGPUNN_SoftMax_updateOutput(input._p, self.output._p)
        return self.output

    def updateGradInput(self, input, gradOutput):
        lib().THGPUNN_SoftMax_updateGradInput(input._p, gradOutput._p, self.gradInput._p, self.output._p)
        return self.gradInput


class SpatialAveragePooling(Module):
    """mcw_nn/SpatialAveragePooling.lua:3-20 (dW, dH default to 1; the output is the window sum, as in the reference)."""

    def __init__(self, kW, kH, dW=1, dH=1):
        super().__init__()
        self.kW, self.kH, self.dW, self.dH = kW, kH, dW, dH

    def updateOutput(self, input):
        _need_gpu(input, "SpatialAveragePooling")
        lib().THGPUNN_SpatialAveragePooling_updateOutput(input._p, self.output._p, self.kW, self.kH, self.dW, self.dH)
        return self.output

    def updateGradInput(self, input, gradOutput):
        if self.gradInput is None:
            return None
        lib().THGPUNN_SpatialAveragePooling_updateGradInput(input._p, gradOutput._p, self.gradInput._p, self.kW, self.kH,
                                                            self.dW, self.dH)
        return self.gradInput


class ClassNLLCriterion:
    """mcw_nn/ClassNLLCriterion.lua GPU branch (:13-19, :42-50): targets are a GPU tensor of 1-based ids."""

    def __init__(self):
        self.sizeAverage = True
        self.outputTensor = GPUTensor(1)
        self.gradInput = GPUTensor()
        self.output = 0.0

    def updateOutput(self, input, target, read_back=True):
        lib().THGPUNN_ClassNLLCriterion_updateOutput(input._p, target._p, self.outputTensor._p, int(self.sizeAverage))
        if read_back:
            self.output = float(self.outputTensor.float()[0])
        return self.output

    forward = updateOutput

    def updateGradInput(self, input, target):
        lib().THGPUNN_ClassNLLCriterion_updateGradInput(input._p, target._p, self.gradInput._p, int(self.sizeAverage))
        return self.gradInput

    backward = updateGradInput
