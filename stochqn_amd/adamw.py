"""First-order steps over the tensors of a model: AdamW with its moments in 32 or in 8 bits, and the norm of all gradients.

The object mirrors the free-mode optimisers of `free.py` -- the caller computes gradients, hands them over with `update_gradient` and
asks for a step with `run_optimizer(step_size)` -- for parameters that are many tensors (f32, bf16, f16) instead of one flat vector.
The arithmetic is the library's (include/stochqn_hip.h, "first-order steps"); all of it runs on the current torch stream, in order
with it, without a synchronisation, and may be captured into a graph.
"""
import ctypes as C
import math

import torch

BLOCK = 128                     # elements that share a scale; every tensor's state starts at a multiple of it


class _Setup(C.Structure):
    _fields_ = [("beta1", C.c_double), ("beta2", C.c_double), ("eps", C.c_double), ("weight_decay", C.c_double),
                ("state_bits", C.c_int), ("stochastic", C.c_int), ("seed", C.c_ulonglong), ("decay", C.c_char_p),
                ("master", C.c_void_p), ("m", C.c_void_p), ("v", C.c_void_p), ("m_scale", C.c_void_p), ("v_scale", C.c_void_p),
                ("count", C.c_void_p), ("work", C.c_void_p)]


_lib = None


def _library():
    global _lib
    if _lib is None:
        from . import cdll
        h = cdll()
        vp, pp, sz, d, i = C.c_void_p, C.POINTER(C.c_void_p), C.c_size_t, C.c_double, C.c_int
        for name, result, args in (
                ("stochqn_hip_tensors_create", vp, [i, pp, C.POINTER(sz), C.POINTER(i)]),
                ("stochqn_hip_tensors_rebind", i, [vp, pp]),
                ("stochqn_hip_tensors_destroy", None, [vp]),
                ("stochqn_hip_tensors_state", sz, [vp, C.POINTER(sz)]),
                ("stochqn_hip_tensors_norm_work", sz, [vp]),
                ("stochqn_hip_tensors_norm", i, [vp, d, d, vp, vp, vp]),
                ("stochqn_hip_adamw_create", vp, [vp, C.POINTER(_Setup)]),
                ("stochqn_hip_adamw_step", i, [vp, vp, d, vp, vp, vp]),
                ("stochqn_hip_adamw_destroy", None, [vp])):
            f = getattr(h, name)
            f.restype, f.argtypes = result, args
        _lib = h
    return _lib


def _types():
    return {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _stream(index):
    """The current torch stream of a device, as the address that the library takes."""
    return torch.cuda.current_stream(index).cuda_stream


# the same without the 2 us that an object for the stream takes
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _stream)


def _scalar(t, device, what):
    """Address of a device tensor of one float32 (None: none)."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.numel() != 1 or t.device != device or t.is_neg():
        raise ValueError("'%s' has to be a float32 tensor of one element on %s." % (what, device))
    return t.data_ptr()


class TensorList:
    """Tensors of one device (parameters, or their gradients) as the library takes them: contiguous, float32 / bfloat16 / float16 each.

    The list keeps the tensors and their memory alive.  `rebind(tensors)` names other ones of the same sizes and types; a graph that was
    captured before goes on with those it saw, which have to be kept alive for it."""

    _handle = None

    def __init__(self, tensors):
        self.tensors = list(tensors)
        types = _types()
        if not self.tensors:
            raise ValueError("no tensors.")
        if not all(getattr(t, "dtype", None) in types for t in self.tensors):
            raise ValueError("tensors have to be float32, bfloat16 or float16.")
        if not self.tensors[0].is_cuda:
            raise ValueError("tensors have to be on one GPU.")
        n = len(self.tensors)
        self.device = self.tensors[0].device
        self._index = self.tensors[0].get_device()
        self.sizes = [t.numel() for t in self.tensors]
        self.dtypes = [t.dtype for t in self.tensors]
        self._at = self._addresses(self.tensors)
        self._memory = [t.untyped_storage() for t in self.tensors]       # a tensor that is given other memory (`.data = ...`) lets go of it
        self._lib = _library()
        with torch.cuda.device(self._index):            # where a list of empty tensors alone belongs
            self._handle = self._lib.stochqn_hip_tensors_create(n, (C.c_void_p * n)(*self._at), (C.c_size_t * n)(*self.sizes),
                                                                (C.c_int * n)(*[types[d] for d in self.dtypes]))
        if not self._handle:
            raise ValueError("the library refused the tensors (its reason is on stderr).")
        self._work = self._lib.stochqn_hip_tensors_norm_work(self._handle)

    def _addresses(self, tensors):
        at = []
        for t, n, dtype in zip(tensors, self.sizes, self.dtypes):
            if getattr(t, "dtype", None) != dtype or t.numel() != n:
                raise ValueError("the tensors have other sizes or types than the list's.")
            if t.get_device() != self._index:
                raise ValueError("tensors have to be on one GPU.")
            if t.layout != torch.strided or not t.is_contiguous() or t.is_neg():
                raise ValueError("tensors have to be dense and contiguous, and no views that negate.")
            at.append(t.data_ptr())
        return at

    def rebind(self, tensors):
        """Other tensors of the same sizes and types take the place of the list's (new gradients of the same parameters)."""
        tensors = list(tensors)
        if len(tensors) != len(self.sizes):
            raise ValueError("the tensors have other sizes or types than the list's.")
        at = self._addresses(tensors)
        if at != self._at:
            if self._lib.stochqn_hip_tensors_rebind(self._handle, (C.c_void_p * len(at))(*at)) != 0:
                raise ValueError("the library refused the tensors (its reason is on stderr).")
            self._at = at
            self._memory = [t.untyped_storage() for t in tensors]
        self.tensors = tensors

    def __len__(self):
        return len(self.tensors)

    def __getstate__(self):
        raise TypeError("a TensorList holds a handle of the library: make a new one of the tensors")

    def norm(self, max_norm=None, grad_scale=1.0, out=None):
        """A float32 tensor of two elements on the device: the norm over all tensors times `grad_scale` (1 / loss scale), and the factor
        that brings the gradients to a norm of at most `max_norm` -- NaN if the norm is not finite as a float32, which makes the step that takes it
        (`run_optimizer(..., grad_scale=out[1:])`) a rejected one.  With a communicator installed: over all ranks' tensors."""
        max_norm = math.inf if max_norm is None else float(max_norm)
        if not max_norm > 0 or not math.isfinite(grad_scale):
            raise ValueError("'max_norm' has to be positive and 'grad_scale' finite.")
        mine = out is None
        if mine:
            out = torch.empty(2, dtype=torch.float32, device=self.device)
        elif (not isinstance(out, torch.Tensor) or out.dtype != torch.float32 or out.shape != (2,) or out.device != self.device
              or out.layout != torch.strided or not out.is_contiguous() or out.is_neg() or out.requires_grad):
            raise ValueError("'out' has to be a float32 tensor of two elements on %s, of which no gradient is taken." % self.device)
        work = torch.empty(self._work, dtype=torch.float64, device=self.device)      # of this call alone: two streams, or two graphs, share none
        if self._lib.stochqn_hip_tensors_norm(self._handle, grad_scale, max_norm, out.data_ptr(), work.data_ptr(), _stream(self._index)) != 0:
            raise RuntimeError("stochqn_hip_tensors_norm failed (its reason is on stderr).")
        if not mine and not out.is_inference():
            torch.autograd.graph.increment_version(out)
        return out

    def __del__(self):
        if self._handle:
            self._lib.stochqn_hip_tensors_destroy(self._handle)


class AdamW_free:
    """AdamW, free mode, over a list of tensors.

    params         tensors (or a TensorList): float32, bfloat16, float16, mixed as they come; updated in place
    state_bits     32: the moments `m`, `v` are float32; 8: float8_e4m3fn / float8_e5m2 codes over float8_e8m0fnu scales of 128
                   elements (`m_scale`, `v_scale`), rounded stochastically
    master         keep float32 weights (`master`) for the 16-bit parameters and take the step on those
    stochastic     without master: round bfloat16 parameters stochastically (no float16 parameters then)
    decay          one truth value per tensor: False = no weight decay for it (biases, norms); None: all decay
    The state is flat tensors of `sum(ceil(n / 128) * 128)` elements; tensor i's begins at `offsets[i]`; `count[0]` is the number of steps.
    """

    _handle = None

    def __init__(self, params, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01, state_bits=32, master=False, stochastic=False,
                 decay=None, seed=0):
        assert 0 <= beta1 < 1 and 0 <= beta2 < 1
        assert 2.0 ** -126 <= eps <= 2.0 ** 126 and math.isfinite(weight_decay)
        assert state_bits in (8, 32)
        assert not (master and stochastic)
        self.params = params if isinstance(params, TensorList) else TensorList(params)
        self.tensors = list(self.params.tensors)        # what the steps write, whatever the list is rebound to later
        self._at, self._memory = list(self.params._at), list(self.params._memory)
        assert not (stochastic and torch.float16 in self.params.dtypes)
        if decay is not None and len(decay) != len(self.params):
            raise ValueError("'decay' has to have one truth value per tensor.")
        self.beta1, self.beta2, self.eps, self.weight_decay = float(beta1), float(beta2), float(eps), float(weight_decay)
        self.state_bits, self.stochastic, self.seed = int(state_bits), bool(stochastic), int(seed) % 2 ** 64
        self.decay = None if decay is None else [bool(d) for d in decay]
        self._lib = _library()
        dev = self.params.device
        offsets = (C.c_size_t * len(self.params))()
        total = self._lib.stochqn_hip_tensors_state(self.params._handle, offsets)
        self.offsets = list(offsets)
        zeros = lambda n, dtype: torch.zeros(n, dtype=dtype, device=dev)
        if self.state_bits == 32:
            self.m, self.v = zeros(total, torch.float32), zeros(total, torch.float32)
            self.m_scale = self.v_scale = None
        else:
            byte = lambda n, dtype: zeros(n, torch.uint8).view(dtype)
            self.m, self.v = byte(total, torch.float8_e4m3fn), byte(total, torch.float8_e5m2)
            self.m_scale, self.v_scale = byte(total // BLOCK, torch.float8_e8m0fnu), byte(total // BLOCK, torch.float8_e8m0fnu)
        self.count, self._work = zeros(2, torch.int64), zeros(512, torch.int64)
        self.master = None
        if master:
            self.master = zeros(total, torch.float32)
            for t, at in zip(self.tensors, self.offsets):
                self.master[at:at + t.numel()].copy_(t.detach().reshape(-1))
        ptr = lambda t: None if t is None else t.data_ptr()
        setup = _Setup(self.beta1, self.beta2, self.eps, self.weight_decay, self.state_bits, int(self.stochastic), self.seed,
                       None if decay is None else bytes(self.decay), ptr(self.master), ptr(self.m), ptr(self.v), ptr(self.m_scale),
                       ptr(self.v_scale), ptr(self.count), ptr(self._work))
        self._handle = self._lib.stochqn_hip_adamw_create(self.params._handle, C.byref(setup))
        if not self._handle:
            raise ValueError("the library refused the optimizer (its reason is on stderr).")
        # The state is complete when the object is there, whichever stream the steps will use ...
        self._on = _stream(dev.index)
        if not torch.cuda.is_current_stream_capturing():
            torch.cuda.current_stream(dev).synchronize()
        self._streams = {self._on}
        self._versioned = [t for t in self.tensors if not t.is_inference()]
        self.gradient = None
        self._own_list = False          # `gradient` was made here, so its tensors may be exchanged here

    def update_gradient(self, gradient):
        """Name the gradients of the coming steps: tensors (or a TensorList) in the order of the parameters.  Nothing is copied: the steps
        read what the tensors hold by then, and they are held until others are named.  None lets go of them, so that a backward pass which makes
        new ones does not find the old ones beside it.  The parameters have to be where they were when the object was made (no `.data = ...`)."""
        if gradient is None:
            self.gradient, self._own_list = None, False
            return
        if [t.data_ptr() for t in self.tensors] != self._at:
            raise ValueError("a parameter has other memory than when the optimizer was made: make a new one, with the old one's state.")
        if isinstance(gradient, TensorList):
            if gradient.sizes != self.params.sizes or gradient.device != self.params.device:
                raise ValueError("the gradients have other sizes or another device than the parameters.")
            self.gradient, self._own_list = gradient, False
            return
        gradient = list(gradient)
        if self._own_list and self.gradient is not None and [getattr(t, "dtype", None) for t in gradient] == self.gradient.dtypes:
            self.gradient.rebind(gradient)
            return
        new = TensorList(gradient)
        if new.sizes != self.params.sizes or new.device != self.params.device:
            raise ValueError("the gradients have other sizes or another device than the parameters.")
        self.gradient, self._own_list = new, True

    def run_optimizer(self, step_size, grad_scale=None):
        """One step.  step_size: a number, or a float32 tensor of one element on the device (schedules in a captured graph).  grad_scale: None,
        or such a tensor that every gradient is multiplied with (`TensorList.norm(...)[1:]`).  If either is not finite (or
        step_size / (1 - beta1 ** t), or step_size * weight_decay, is past float32) the step is rejected: no weight, no moment and no count changes."""
        gradient = self.gradient                        # this step's, also if another thread names others meanwhile
        if gradient is None:
            raise ValueError("no gradient: call update_gradient first.")
        dev = self.params.device
        step_dev = None
        if isinstance(step_size, torch.Tensor):
            step_dev, step_size = _scalar(step_size, dev, "step_size"), 0.0
        elif not math.isfinite(step_size):
            raise ValueError("'step_size' is not finite.")
        scale = _scalar(grad_scale, dev, "grad_scale")
        stream = _stream(dev.index)
        if stream != self._on:
            self._used_on(stream)
        if self._lib.stochqn_hip_adamw_step(self._handle, gradient._handle, step_size, step_dev, scale, stream) != 0:
            raise RuntimeError("stochqn_hip_adamw_step failed (its reason is on stderr).")
        torch.autograd.graph.increment_version(self._versioned)          # a graph that saved the old weights cannot be run backward any more

    def _used_on(self, stream):
        """... and its memory is not given to others before the work of those streams is done.  A capture runs nothing: the stream that it is made
        on is still to be recorded at its first step outside of one."""
        if stream not in self._streams:
            if torch.cuda.is_current_stream_capturing():
                return
            self._streams.add(stream)
            for t in (self.m, self.v, self.m_scale, self.v_scale, self.master, self.count, self._work):
                if t is not None:
                    t.record_stream(torch.cuda.current_stream(self.params.device))
        self._on = stream

    def __getstate__(self):
        raise TypeError("an AdamW_free holds a handle of the library: carry its state_dict() instead")

    def moments(self, i):
        """The two moments of tensor i as float32, in its shape (copies for 8-bit moments, views otherwise)."""
        t, at = self.tensors[i], self.offsets[i]
        out = []
        for x, by in ((self.m, self.m_scale), (self.v, self.v_scale)):
            if by is not None:
                upto = at + -(-t.numel() // BLOCK) * BLOCK
                x = (x[at:upto].float().view(-1, BLOCK) * by[at // BLOCK:upto // BLOCK].float()[:, None]).view(-1)
                out.append(x[:t.numel()].view(t.shape))
            else:
                out.append(x[at:at + t.numel()].view(t.shape))
        return tuple(out)

    def state_dict(self):
        """The state (references, not copies) and the numbers that the steps were taken with."""
        names = ("m", "v", "m_scale", "v_scale", "master", "count")
        state = {k: getattr(self, k) for k in names if getattr(self, k) is not None}
        return dict(state, beta1=self.beta1, beta2=self.beta2, eps=self.eps, weight_decay=self.weight_decay, state_bits=self.state_bits,
                    stochastic=self.stochastic, seed=self.seed, decay=self.decay, sizes=list(self.params.sizes))

    def load_state_dict(self, state):
        """Take over the state of another object over tensors of the same sizes, constructed with the same numbers."""
        mine = self.state_dict()
        same = ("beta1", "beta2", "eps", "weight_decay", "state_bits", "stochastic", "seed", "decay", "sizes")
        if set(state) != set(mine) or any(state[k] != mine[k] for k in same):
            raise ValueError("the state belongs to an optimizer that was constructed otherwise.")
        arrays = set(mine) - set(same)
        if any(getattr(state[k], "shape", None) != mine[k].shape or state[k].dtype != mine[k].dtype for k in arrays):
            raise ValueError("the state's arrays have other shapes or types than this optimizer's.")
        for k in arrays:
            mine[k].copy_(state[k])

    def __del__(self):
        if self._handle:
            self._lib.stochqn_hip_adamw_destroy(self._handle)
