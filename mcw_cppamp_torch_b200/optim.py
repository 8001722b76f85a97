"""Parameter updates that keep a state of their own, over the tensors of `Module.parameters()` or `getParameters()`."""
from ._lib import TP, lib
from .tensor import GPUTensor

BLOCK = 256     # values under one scale of the 8-bit moments


def _tensors(t, what):
    t = [t] if isinstance(t, GPUTensor) else list(t)
    for v in t:
        if not isinstance(v, GPUTensor):
            raise TypeError("%s: torch.GPUTensor expected (call :gpu() on the module first)" % what)
    return t


class AdamW:
    """Adam with decoupled weight decay: update() takes a step of all `weights` by their `gradWeights`, tensors or lists of them as
    `net.parameters()` and `net.getParameters()` give, in one launch.

        opt = gt.optim.AdamW(*net.getParameters(), learningRate=1e-3)
        net.zeroGradParameters(); net.backward(...); opt.update()

    bits=32: the moments lie in `mean` and `square`, a tensor for each of the weights.  bits=8: in `meanCodes`, `rootCodes` and `scales`, 2.03 bytes a value
    instead of 8, rounded at random by `seed`; moments() gives what they stand for.  `step` holds the number of steps taken, on the device (up to 2^24), so that a
    recorded update counts on when it is replayed; learningRate and the others are those of the recording.  Gradients may share memory, what a step writes may not."""

    def __init__(self, weights, gradWeights, learningRate=1e-3, beta1=0.9, beta2=0.999, epsilon=1e-8, weightDecay=0.01, bits=32, seed=0):
        self.weights, self.gradWeights = _tensors(weights, "AdamW"), _tensors(gradWeights, "AdamW gradients")
        if len(self.weights) != len(self.gradWeights):
            raise ValueError("AdamW: a gradient for each tensor expected")
        if bits not in (8, 32):
            raise ValueError("AdamW: moments are held in 8 or in 32 bits")
        self.learningRate, self.beta1, self.beta2, self.epsilon, self.weightDecay = learningRate, beta1, beta2, epsilon, weightDecay
        self.bits, self.seed = bits, seed
        self._arrays = {}
        self.step = GPUTensor(2).zero()
        if bits == 32:
            self.mean, self.square = ([_zeros(*w.size()) for w in self.weights] for _ in range(2))
        else:
            blocks = [-(-w.nElement() // BLOCK) for w in self.weights]
            self.meanCodes, self.rootCodes = ([_zeros(b * BLOCK // 4) for b in blocks] for _ in range(2))
            self.scales = [_zeros(2 * b) for b in blocks]

    def _array(self, name, tensors):
        """The tensors as the library takes them, made again when others have come to the list."""
        if len(tensors) != len(self.weights):
            raise ValueError("AdamW: a tensor of each kind for each of the weights expected")
        held, array = self._arrays.get(name, (None, None))
        if held != tensors:
            held = list(tensors)
            array = (TP * max(1, len(held)))(*[t._p for t in held])
            self._arrays[name] = held, array
        return array

    def __getstate__(self):
        return dict(self.__dict__, _arrays={})

    def update(self):
        names = ("weights", "gradWeights") + (("mean", "square") if self.bits == 32 else ("meanCodes", "rootCodes", "scales"))
        call = (len(self.weights),) + tuple(self._array(n, getattr(self, n)) for n in names)
        call += (self.step._p, float(self.learningRate), float(self.beta1), float(self.beta2), float(self.epsilon), float(self.weightDecay))
        if self.bits == 32:
            lib().THGPUNN_AdamW_update(*call)
        else:
            lib().THGPUNN_AdamW8_update(*call, int(self.seed))

    def moments(self, mean=None, square=None):
        """The moments as lists of tensors: those that update() keeps, or with 8 bits what their codes stand for, in `mean` and `square` where these are given."""
        if self.bits == 32:
            if mean is not None or square is not None:
                raise ValueError("AdamW: moments of 32 bits are not copied")
            return self.mean, self.square
        mean, square = ([GPUTensor(*w.size()) for w in self.weights] if t is None else _tensors(t, "AdamW moments") for t in (mean, square))
        lists = [self._array(n, getattr(self, n)) for n in ("meanCodes", "rootCodes", "scales")] + [self._array("mean", mean), self._array("square", square)]
        lib().THGPUNN_AdamW8_moments(len(self.weights), *lists)
        return mean, square


def _zeros(*sizes):
    return GPUTensor(*sizes).zero() if sizes and min(sizes) else GPUTensor()
