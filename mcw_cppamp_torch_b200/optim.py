"""Parameter updates that keep a state of their own, over the parameters of modules."""
from . import _lib
from ._lib import TP, lib
from .tensor import GPUTensor

BLOCK = 256     # values under one scale of the 8-bit moments
# The rounding noise of 8-bit moments is a hash of (seed ^ step * odd number) + place * the same number: with the seed 0 a place's noise is that of its neighbour a step later, with
# other seeds of few bits some steps later.  Of this one (digits of e), in a million steps, no two that are up to eight apart have the same noise less than a million places apart.
SEED = 0xb7e15163


def parameters(*modules):
    """The weights and the gradients of modules, and of those that containers hold, as two lists."""
    weights, gradients = [], []
    for module in modules:
        for m in module.modules_list():
            w, g = m.parameters() or ([], [])
            weights += w
            gradients += g
    return weights, gradients


def _array(tensors, what):
    """One tensor or several as a tuple, and the array of their pointers that the library takes, which the tuple has to outlive."""
    tensors = (tensors,) if isinstance(tensors, GPUTensor) else tuple(tensors)
    lib()
    try:
        pointers = _lib.calls.pointers(tensors)
    except TypeError as e:
        raise TypeError("AdamW %s: %s (call :gpu() on the module first)" % (what, e)) from None
    return tensors, (TP * max(1, len(tensors))).from_buffer(pointers)


def _once(weights, gradients):
    """Each of the weights once, by its memory, with its gradient: a module that occurs several times lists its tensors as often."""
    seen, kept = {}, []
    for i, (w, g) in enumerate(zip(weights, gradients)):
        at, n = w.data_ptr(), w.nElement()
        first, gradient = seen.setdefault((at, n), (i, g.data_ptr())) if n else (i, None)
        if first == i:
            kept.append(i)
        elif gradient != g.data_ptr():
            raise ValueError("AdamW: tensors %d and %d are the same weights, with two gradients" % (first + 1, i + 1))
    return tuple(weights[i] for i in kept), tuple(gradients[i] for i in kept)


class _Tensors:
    """A sequence of tensors as a field: kept as a tuple, so that the array of them that the library takes is made once for each that is put there."""

    def __set_name__(self, owner, name):
        self.name = name

    def __get__(self, obj, owner=None):
        if obj is None:
            return self
        if self.name not in obj._lists:      # the other width's moments
            raise AttributeError("AdamW: no %s among the tensors of this one" % self.name)
        return obj._lists[self.name][0]

    def __set__(self, obj, tensors):
        obj._lists[self.name] = _array(tensors, self.name)


class AdamW:
    """Adam with decoupled weight decay: update() takes a step of all `weights` by their `gradWeights`, tensors or lists of them as `parameters(net)` and
    `net.getParameters()` give, in one launch.

        opt = gt.optim.AdamW(*gt.optim.parameters(net), learningRate=1e-3)
        net.zeroGradParameters(); net.backward(...); opt.update()

    bits=32: the moments lie in `mean` and `square`, a tensor for each of the weights.  bits=8: in `meanCodes`, `rootCodes` and `scales`, 2.03 bytes a value
    instead of 8, rounded at random by `seed` (a word with many bits set: see SEED); moments() gives what they stand for.  `step` holds the number of steps taken, on the device (up to 2^24), so that a
    recorded update counts on when it is replayed; learningRate and the others are those of the recording.  Weights that are listed again, as those of a module that occurs twice,
    are updated once.  Gradients may share memory, what a step writes may not.
    Saved along with its module, gt.save([net, opt], path), it has the module's tensors again after loading."""

    weights, gradWeights, mean, square, meanCodes, rootCodes, scales = (_Tensors() for _ in range(7))      # tuples: a list put there becomes one

    def __init__(self, weights, gradWeights, learningRate=1e-3, beta1=0.9, beta2=0.999, epsilon=1e-8, weightDecay=0.01, bits=32, seed=SEED):
        self._lists = {}
        self.weights, self.gradWeights = weights, gradWeights
        if len(self.weights) != len(self.gradWeights):
            raise ValueError("AdamW: a gradient for each tensor expected")
        once = _once(self.weights, self.gradWeights)
        if len(once[0]) < len(self.weights):
            self.weights, self.gradWeights = once
        if bits not in (8, 32):
            raise ValueError("AdamW: moments are held in 8 or in 32 bits")
        self.learningRate, self.beta1, self.beta2, self.epsilon, self.weightDecay = learningRate, beta1, beta2, epsilon, weightDecay
        self.bits, self.seed = bits, seed
        self.step = GPUTensor(2).zero()
        if bits == 32:
            self.mean, self.square = ([_zeros(*w.size()) for w in self.weights] for _ in range(2))
        else:
            blocks = [-(-w.nElement() // BLOCK) for w in self.weights]
            self.meanCodes, self.rootCodes = ([_zeros(b * BLOCK // 4) for b in blocks] for _ in range(2))
            self.scales = [_zeros(2 * b) for b in blocks]

    def _arrays(self, *names):
        if any(len(self._lists[n][0]) != len(self.weights) for n in names):
            raise ValueError("AdamW: a tensor of each kind for each of the weights expected")
        return [self._lists[n][1] for n in names]

    def __getstate__(self):
        return dict(self.__dict__, _lists={n: t for n, (t, _) in self._lists.items()})

    def __setstate__(self, state):
        self.__dict__.update(state, _lists={})
        for n, t in state["_lists"].items():
            setattr(self, n, t)

    def update(self):
        rates = (self.step._p, float(self.learningRate), float(self.beta1), float(self.beta2), float(self.epsilon), float(self.weightDecay))
        if self.bits == 32:
            lib().THGPUNN_AdamW_update(len(self.weights), *self._arrays("weights", "gradWeights", "mean", "square"), *rates)
        else:
            lib().THGPUNN_AdamW8_update(len(self.weights), *self._arrays("weights", "gradWeights", "meanCodes", "rootCodes", "scales"), *rates, int(self.seed))

    def moments(self, mean=None, square=None):
        """The moments as lists of tensors: those that update() keeps, or with 8 bits what their codes stand for, in `mean` and `square` where these are given."""
        if self.bits == 32:
            if mean is not None or square is not None:
                raise ValueError("AdamW: moments of 32 bits are not copied")
            return self.mean, self.square
        (mean, means), (square, squares) = (_array([GPUTensor(*w.size()) for w in self.weights] if t is None else t, "moments") for t in (mean, square))
        if not len(mean) == len(square) == len(self.weights):
            raise ValueError("AdamW: a tensor for each of the weights expected")
        lib().THGPUNN_AdamW8_moments(len(mean), *self._arrays("meanCodes", "rootCodes", "scales"), means, squares)
        return mean, square


def _zeros(*sizes):
    return GPUTensor(*sizes).zero() if sizes and min(sizes) else GPUTensor()
