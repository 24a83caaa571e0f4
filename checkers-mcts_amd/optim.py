"""AdamW over many tensors in one launch, with moments in 32 or in 8 bits (csrc/ckr_adamw.hip).

The reference trains with Keras' Adam (training_pipeline.py:113), which `train_hip.HipTrainStep` has for the 128-kernel network in
float32.  This optimiser takes any module's parameters, in float32, bfloat16 or float16; `train.train_nn` uses it under OPTIMIZER.
"""
import ctypes as C
import math
from array import array
from operator import attrgetter

import torch

from . import _lib

BLOCK = 128                         # elements that share a scale in 8-bit moments; every tensor's part of the states is padded to it
TENSORS, BLOCKS = 128, 2048         # of one launch (ckr_adamw.hip)
TICKET_WORDS = 1056                 # CKR_TICKET_WORDS
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
# accessors for map(): a step looks at every parameter and gradient
_SHAPE, _DTYPE, _GRAD, _NBYTES = attrgetter("shape"), attrgetter("dtype"), attrgetter("grad"), attrgetter("nbytes")
_VERSION = attrgetter("_version")
_STRIDE, _DEVICE, _POINTER = torch.Tensor.stride, torch.Tensor.get_device, torch.Tensor.data_ptr
_NEGATED = torch.Tensor.is_neg      # memory that holds the opposite sign: the gradient of an imaginary part, of one element, may come so


def _guards():
    """torch's native comparison of many tensors' types, devices, sizes and strides with those of examples, if it sees all that matters
    here: one call instead of six map()s over the parameters (a step of 170 tensors, wall time: 79 us, 97 us with the map()s)."""
    try:
        from torch._C._dynamo.guards import TensorGuards
        x = torch.zeros((4, 4), dtype=torch.float16)
        make = lambda *tensors: TensorGuards(*tensors, dynamic_dims_sizes=None, dynamic_dims_strides=None)
        g, row = make(x, x), make(x[0])
        others = (x.t(), x[:2], x.view(torch.bfloat16), x.view(torch.int16), x.to("meta"), x.reshape(2, 8), x[None], torch._neg_view(x), x.to_sparse(), None)
        if g.check(x, torch.ones_like(x)) and row.check(x[1]) and not row.check(x[:, 0]) and not any(g.check(x, y) or g.check(y, x) for y in others):
            return make
    except Exception:                                                  # (not a public name: another torch may not have it, or in another form)
        pass
    return None


_make_guards = _guards()


class AdamWArgs(C.Structure):
    """ckr_adamw_args (include/ckr.h)."""
    _fields_ = [(n, C.c_void_p) for n in ("sizes", "offsets", "params", "grads", "master", "m", "v", "m_scale", "v_scale",
                                          "d_step", "d_ticket", "d_lr", "d_norm")] + \
        [(n, C.c_double) for n in ("lr", "beta1", "beta2", "weight_decay")] + [("seed", C.c_uint64), ("eps", C.c_float)] + \
        [(n, C.c_int32) for n in ("count", "dtype", "state_bits")]


def _layout(t):
    """Strides of the dimensions that have more than one element; None unless the tensor fills its memory without gaps or overlaps."""
    dims = [(st, n) for n, st in zip(t.shape, t.stride()) if n > 1]
    want = 1
    for st, n in sorted(dims):
        if st != want:
            return None
        want *= n
    return dims


class _Batch:
    """The tensors of one group and type: what one call of ckr_adamw_step takes."""

    def __init__(self, group, dtype, params, offsets, first):
        self.group, self.dtype, self.params, self.first, self.n = group, dtype, params, first, len(params)
        self.sizes = (C.c_int64 * self.n)(*[p.numel() for p in params])
        self.offsets = (C.c_int64 * self.n)(*offsets)
        self.seen = None                                               # the group's hyperparameters that passed the checks last


class AdamW:
    """AdamW with decoupled weight decay:

        m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;  w = w (1 - lr weight_decay) - lr m^ / (sqrt(v^) + eps)

    with m^, v^ the bias-corrected moments and every tensor's own step count (a tensor without a gradient is left alone).

    params        tensors, or groups {"params": [...], "lr": ..., "betas": ..., "eps": ..., "weight_decay": ...}, of float32, bfloat16
                  or float16 on one GPU, dense in memory (any order of dimensions).  16-bit parameters get a float32 master copy, which is
                  what the optimiser updates; the parameter is its rounding, and where something else has changed it, the copy follows
                  (reset_master()).  Their memory may be replaced (p.data = ...) by some of the same shape, strides and type.
    lr            a number, or a float32 device scalar (read by the kernel: a captured step follows its changes).
    state_bits    32, or 8: a byte for each moment and a scale byte for each 128 elements, rounded stochastically (seed).
    max_norm      clip the gradients by their global norm (over all groups): g * min(1, max_norm / (norm + 1e-6)); the norm of the last
                  step is `grad_norm`, a float64 device scalar.

    It is no torch.optim.Optimizer, which torch.optim.lr_scheduler asks for: a schedule sets param_groups[i]["lr"] or fills the device scalar.
    step() runs on the current stream and does not synchronise; it can be captured into a HIP graph (gradients then have to stay where
    they are: zero_grad(set_to_none=False)).  Steps of one optimiser must not run at the same time."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, max_norm=None, seed=0):
        if state_bits not in (32, 8):
            raise ValueError("state_bits must be 32 or 8, got %r" % (state_bits,))
        if max_norm is not None and not (0 < float(max_norm) < math.inf):
            raise ValueError("max_norm must be positive and finite, got %r" % (max_norm,))
        if isinstance(params, torch.Tensor):
            raise ValueError("params must be a list of tensors or of groups, got a tensor")
        params = list(params)
        groups = [dict(g) for g in params] if params and isinstance(params[0], dict) else [{"params": params}]
        for g in groups:
            g["params"] = [g["params"]] if isinstance(g["params"], torch.Tensor) else list(g["params"])
            for k, dflt in (("lr", lr), ("betas", betas), ("eps", eps), ("weight_decay", weight_decay)):
                g.setdefault(k, dflt)
        self.param_groups, self.state_bits, self._max_norm, self.seed = groups, int(state_bits), None if max_norm is None else float(max_norm), int(seed) & (2 ** 64 - 1)
        every = [p for g in groups for p in g["params"]]
        if not every:
            raise ValueError("AdamW: no parameters")
        for p in every:
            if not isinstance(p, torch.Tensor) or not p.is_cuda or p.dtype not in DTYPES or p.device != every[0].device:
                raise ValueError("parameters must be float32, bfloat16 or float16 tensors on one GPU")
            if not p.is_leaf:
                raise ValueError("AdamW steps leaf tensors only")
            if p.is_neg():
                raise ValueError("a parameter is a view of the negative of its memory")
            if _layout(p) is None:
                raise ValueError("a parameter of shape %s and strides %s does not fill its memory" % (list(p.shape), list(p.stride())))
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in every if p.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("parameters share memory (or one is listed twice)")
        self.device = dev = every[0].device
        for g in groups:
            self._check_group(g)
        # the states: one flat buffer a moment, tensor i at offsets[i]
        self.params, self.offsets, total = every, [], 0
        for p in every:
            self.offsets.append(total)
            total += (p.numel() + BLOCK - 1) // BLOCK * BLOCK
        self.total = total
        where = {id(p): o for p, o in zip(every, self.offsets)}
        self._batches, first = [], 0
        for g in groups:
            for dtype in DTYPES:
                mine = [p for p in g["params"] if p.dtype == dtype and p.numel()]
                if mine:
                    self._batches.append(_Batch(g, dtype, mine, [where[id(p)] for p in mine], first))
                    first += len(mine)
        state = torch.uint8 if self.state_bits == 8 else torch.float32
        z = lambda n, dtype: torch.zeros((n,), dtype=dtype, device=dev)
        self.exp_avg, self.exp_avg_sq = z(total, state), z(total, state)
        self.scales = (torch.ones((2, max(1, total // BLOCK)), dtype=torch.uint8, device=dev)) if self.state_bits == 8 else None
        self._every = [p for b in self._batches for p in b.params]     # in the order of the batches
        self._half = [i for i, p in enumerate(self._every) if p.dtype != torch.float32]
        self._half_params = [self._every[i] for i in self._half]
        self.master, self._versions = None, []
        if any(p.dtype != torch.float32 for p in every):
            self.master = z(total, torch.float32)
            self.reset_master()
        self.steps = z(max(1, first), torch.int32)                     # in the order of the batches
        self._ticket = z(2 * TICKET_WORDS, torch.int32)                # of the step, of the norm
        # partial sums of the norm: one launch for each run of up to TENSORS tensors of one type
        launches = sum((b.n + TENSORS - 1) // TENSORS for b in self._batches)
        self._parts, self._norm = (z(max(1, launches) * BLOCKS, torch.float64), z(2, torch.float64)) if self._max_norm is not None else (None, None)
        self._sizes_all = (C.c_int64 * first)(*[p.numel() for p in self._every])
        self._dtypes_all = (C.c_int32 * first)(*[DTYPES[p.dtype] for p in self._every])
        self._layouts = [_layout(p) for p in self._every]
        self._shape_of, self._stride_of, self._type_of, self._nbytes_of = ([f(p) for p in self._every] for f in (_SHAPE, _STRIDE, _DTYPE, _NBYTES))
        self._device_of, self._offset_of = [dev.index] * first, [where[id(p)] for p in self._every]
        # what the order of the states follows from: each group's parameters, their types and, where they are not row by row, how they lie
        self._arrangement = [[[str(p.dtype)] + ([] if p.is_contiguous() else [list(n) for n in _layout(p)]) for p in g["params"]] for g in groups]
        self._guards, self._found = None, False                        # of parameters and gradients that were found to be as above
        self._adopt()
        self._streams = {torch.cuda.current_stream(dev).cuda_stream}
        torch.cuda.current_stream(dev).synchronize()                   # a step on any stream finds the states in place
        self._L = _lib.load()
        ptr = lambda t: None if t is None else t.data_ptr()
        scales = (None, None) if self.scales is None else (self.scales[0].data_ptr(), self.scales[1].data_ptr())
        self._states = (ptr(self.master), self.exp_avg.data_ptr(), self.exp_avg_sq.data_ptr()) + scales
        self._steps_ptr, self._ticket_ptr, self._norm_ptr = self.steps.data_ptr(), self._ticket.data_ptr(), ptr(self._norm)

    def _check_group(self, g):
        lr = g["lr"]
        if isinstance(lr, torch.Tensor):
            if lr.device != self.device or lr.dtype != torch.float32 or lr.numel() != 1:
                raise ValueError("lr must be a number or a float32 scalar on %s" % self.device)
        elif not 0 <= float(lr) < math.inf:
            raise ValueError("lr must be finite and not negative, got %r" % (lr,))
        b1, b2 = g["betas"]
        if not (0 <= b1 < 1 and 0 <= b2 < 1):
            raise ValueError("betas must be in [0, 1), got %r" % (g["betas"],))
        if not 1e-37 <= float(g["eps"]) <= 1e30:
            raise ValueError("eps must be positive (1e-37 to 1e30), got %r" % (g["eps"],))
        if not 0 <= float(g["weight_decay"]) < math.inf:
            raise ValueError("weight_decay must be finite and not negative, got %r" % (g["weight_decay"],))

    @staticmethod
    def _flat_view(flat, p, offset):
        """p's part of a flat buffer, in p's own shape and order of dimensions."""
        return flat.as_strided(p.shape, p.stride(), flat.storage_offset() + offset) if p.numel() else flat.new_empty(p.shape)

    def _pointers(self):
        """Device addresses of all parameters and gradients in the order of the batches (0: no gradient), and copies of gradients that lie
        otherwise than their parameters."""
        ps, keep = self._every, []
        addresses = list(map(_POINTER, ps))
        if addresses != self._addresses:                               # (_aliases keep the memory: at the same address it is the same)
            moved = [i for i in self._half if addresses[i] != self._addresses[i]]
            self._adopt()
            self._follow(moved)
            addresses = self._addresses
        if self._half and (versions := list(map(_VERSION, self._half_params))) != self._versions:
            self._follow([i for i, now, then in zip(self._half, versions, self._versions) if now != then])
            self._versions = versions
        gs = list(map(_GRAD, ps))
        if self._guards is not None and self._guards.check(*ps, *gs):
            return array("Q", addresses), array("Q", map(_POINTER, gs)), keep
        if list(map(_STRIDE, ps)) != self._stride_of or list(map(_DTYPE, ps)) != self._type_of:      # the same memory, seen otherwise
            self._adopt()
        try:
            if list(map(_STRIDE, gs)) == self._stride_of and list(map(_DTYPE, gs)) == self._type_of and list(map(_NBYTES, gs)) == self._nbytes_of \
                    and list(map(_DEVICE, gs)) == self._device_of and not any(map(_NEGATED, gs)):
                self._guards = None if _make_guards is None or not self._found else _make_guards(*ps, *gs)      # (made in the second such step)
                self._found = True
                return array("Q", addresses), array("Q", map(_POINTER, gs)), keep
        except (TypeError, AttributeError, RuntimeError):              # None, or sparse
            pass
        gs = [self._gradient(i, g, keep) for i, g in enumerate(gs)]
        return array("Q", addresses), array("Q", (0 if g is None else g.data_ptr() for g in gs)), keep

    def _adopt(self):
        """Takes the parameters' memory as it is now, if it is laid out as it was."""
        for p, shape, stride, dtype in zip(self._every, self._shape_of, self._stride_of, self._type_of):
            if p.shape != shape or p.stride() != stride or p.dtype != dtype or p.device != self.device:
                raise ValueError("a parameter's shape, strides, type or device changed after the optimiser was made")
        self._aliases = [p.detach() for p in self._every]
        self._addresses = list(map(_POINTER, self._every))

    @torch.no_grad()
    def _follow(self, which):
        """Something else than a step has changed these 16-bit parameters: where one is no longer the rounding of its master copy, the copy
        takes its value."""
        for i in which:
            p = self._every[i]
            if p.shape != self._shape_of[i] or p.stride() != self._stride_of[i] or p.dtype != self._type_of[i]:
                raise ValueError("a parameter's shape, strides, type or device changed after the optimiser was made")
            master = self._flat_view(self.master, p, self._offset_of[i])
            master.copy_(torch.where(master.to(p.dtype) == p.detach(), master, p.detach().float()))

    def _gradient(self, i, g, keep):
        if g is None:
            return None
        if g.layout != torch.strided:
            raise ValueError("sparse gradients are not supported")
        if g.shape != self._shape_of[i] or g.dtype != self._type_of[i] or g.device != self.device:
            raise ValueError("a gradient must have its parameter's shape, type and device")
        if _layout(g) != self._layouts[i] or g.is_neg():               # (a copy of a view of the negative holds its values)
            g = torch.empty_strided(g.shape, self._stride_of[i], dtype=g.dtype, device=g.device).copy_(g.detach())
            keep.append(g)
        return g

    def step(self):
        """One update of every parameter that has a gradient."""
        if torch.cuda.current_device() != self.device.index:
            with torch.cuda.device(self.device):
                return self._step()
        return self._step()

    def _step(self):
        L, s = self._L, _lib.raw_stream(self.device.index)
        if s not in self._streams:                                     # the allocator has to know before it hands the memory on
            self._streams.add(s)
            for t in (self.exp_avg, self.exp_avg_sq, self.scales, self.master, self.steps, self._ticket, self._parts, self._norm):
                if t is not None:
                    t.record_stream(torch.cuda.current_stream(self.device))
        for b in self._batches:
            g = b.group
            now = g["lr"], g["betas"], g["eps"], g["weight_decay"]
            if b.seen is None or not all(x is y for x, y in zip(now, b.seen)):
                self._check_group(g)
                b.seen = now
        ps, gs, keep = self._pointers()
        p0, g0 = ps.buffer_info()[0], gs.buffer_info()[0]
        if self._max_norm is not None:
            _lib.check(L.ckr_grad_norm(len(gs), self._sizes_all, g0, self._dtypes_all, self._max_norm, self._parts.data_ptr(), self._parts.numel(),
                                       self._ticket.data_ptr() + 4 * TICKET_WORDS, self._norm.data_ptr(), s))
        for b in self._batches:
            lr, (b1, b2), eps, decay = b.seen
            on_device = isinstance(lr, torch.Tensor)
            a = AdamWArgs(C.addressof(b.sizes), C.addressof(b.offsets), p0 + 8 * b.first, g0 + 8 * b.first, *self._states, self._steps_ptr + 4 * b.first, self._ticket_ptr,
                          lr.data_ptr() if on_device else None, self._norm_ptr, 0.0 if on_device else float(lr), float(b1), float(b2), float(decay), self.seed,
                          float(eps), b.n, DTYPES[b.dtype], self.state_bits)
            _lib.check(L.ckr_adamw_step(C.byref(a), s))
        stepped = self._every if 0 not in gs else [p for p, g in zip(self._every, gs) if g]
        if stepped:
            torch.autograd.graph.increment_version(stepped)            # a backward pass over what it saved before the step is refused
        if self._half:
            self._versions = list(map(_VERSION, self._half_params))    # (views of one buffer share a counter: not simply one more)

    @property
    def max_norm(self):
        return self._max_norm

    @property
    def grad_norm(self):
        """The global norm of the last step's gradients before clipping (float64 device scalar; None without max_norm)."""
        return None if self._norm is None else self._norm[0]

    def zero_grad(self, set_to_none=True):
        grads = [p.grad for p in self.params if p.grad is not None]
        if set_to_none:
            for p in self.params:
                p.grad = None
        elif grads:
            with torch.no_grad():
                torch._foreach_zero_(grads)

    @torch.no_grad()
    def reset_master(self):
        """Takes the master copies from the 16-bit parameters.  step() sees by itself what has changed them in place (load_state_dict() of the
        module, say) or replaced their memory.  What torch's version counters do not show (p.data.copy_(), another replayed graph) it
        would undo, and the replay of a captured step undoes any change: call this first."""
        for p, o in zip(self.params, self.offsets):
            if p.dtype != torch.float32:
                self._flat_view(self.master, p, o).copy_(p.detach())
        self._versions = list(map(_VERSION, self._half_params))

    # ---- states ---------------------------------------------------------------------------------------------
    def moments(self):
        """(m, v) as float32 flat tensors, tensor i at offsets[i] (split() has the views); with 32-bit states the states themselves, with
        8 bits the values that the codes stand for."""
        if self.state_bits == 32:
            return self.exp_avg, self.exp_avg_sq
        m, v = (torch.empty((self.total,), dtype=torch.float32, device=self.device) for _ in range(2))
        if self.total:
            self._on_device(self._L.ckr_adamw_read_moments, *self._states[1:], self.total, m.data_ptr(), v.data_ptr())
        return m, v

    def _on_device(self, fn, *args):
        if torch.cuda.current_device() == self.device.index:
            _lib.check(fn(*args, _lib.raw_stream(self.device.index)))
        else:
            with torch.cuda.device(self.device):
                _lib.check(fn(*args, _lib.raw_stream(self.device.index)))

    def split(self, flat):
        """Views of a flat tensor of moments (or of `master`), one for each parameter, in its shape."""
        return [self._flat_view(flat, p, o) for p, o in zip(self.params, self.offsets)]

    @torch.no_grad()
    def load_moments(self, exp_avg, exp_avg_sq, step):
        """Moments from float32 values (flat, as moments() gives them, or a list of tensors like the parameters) after `step` steps; with 8-bit
        states to the nearest codes."""
        flat = []
        for given in (exp_avg, exp_avg_sq):
            if isinstance(given, torch.Tensor):
                if given.shape != (self.total,) or given.dtype != torch.float32 or given.device != self.device:
                    raise ValueError("moments must be float32 [%d] on %s" % (self.total, self.device))
                flat.append(given.contiguous())
            else:
                given = list(given)
                if len(given) != len(self.params) or any(t.shape != p.shape for t, p in zip(given, self.params)):
                    raise ValueError("moments must have the parameters' shapes")
                buf = torch.zeros((self.total,), dtype=torch.float32, device=self.device)
                for view, t in zip(self.split(buf), given):
                    view.copy_(t)
                flat.append(buf)
        if self.state_bits == 32:
            self.exp_avg.copy_(flat[0])
            self.exp_avg_sq.copy_(flat[1])
        elif self.total:
            self._on_device(self._L.ckr_adamw_write_moments, flat[0].data_ptr(), flat[1].data_ptr(), self.total, *self._states[1:])
        self.steps.fill_(int(step))

    def state_dict(self):
        """States (the buffers themselves) and hyperparameters; load_state_dict() of an optimiser over the same parameters takes it.  The
        parameters are not among them, the master copies of 16-bit ones are."""
        return {"layout": self._arrangement, "state_bits": self.state_bits, "seed": self.seed, "exp_avg": self.exp_avg, "exp_avg_sq": self.exp_avg_sq, "scales": self.scales,
                "master": self.master, "steps": self.steps, "sizes": [p.numel() for p in self.params],
                "param_groups": [{k: v for k, v in g.items() if k != "params"} for g in self.param_groups]}

    @torch.no_grad()
    def load_state_dict(self, state):
        """A learning rate on the device keeps its scalar, which takes the saved value: captured steps go on reading it."""
        if state["state_bits"] != self.state_bits or state["sizes"] != [p.numel() for p in self.params] or len(state["param_groups"]) != len(self.param_groups) \
                or (state["master"] is None) != (self.master is None) or state["steps"].numel() != self.steps.numel():
            raise ValueError("the state belongs to other parameters, groups or state_bits")
        if state.get("layout", self._arrangement) != self._arrangement:     # (states saved before it was among them: as they are)
            raise ValueError("the state belongs to parameters of other types, orders in memory or groups; moments() with split(), and load_moments(), "
                             "carry moments over")
        groups = []
        for g, new in zip(self.param_groups, state["param_groups"]):
            new = dict(new)
            if isinstance(new.get("lr"), torch.Tensor):                # of another device, or another optimiser's own
                new["lr"] = new["lr"].to(self.device, copy=True)
            self._check_group(dict(g, **new))
            groups.append(new)
        for mine, other in ((self.exp_avg, state["exp_avg"]), (self.exp_avg_sq, state["exp_avg_sq"]), (self.scales, state["scales"]),
                            (self.master, state["master"]), (self.steps, state["steps"])):
            if mine is not None:
                mine.copy_(other)
        self._versions = list(map(_VERSION, self._half_params))        # the masters are the state's
        self.seed = state["seed"]
        for g, new in zip(self.param_groups, groups):
            if isinstance(g["lr"], torch.Tensor) and "lr" in new:
                value = new.pop("lr")
                g["lr"].copy_(value.reshape(g["lr"].shape)) if isinstance(value, torch.Tensor) else g["lr"].fill_(float(value))
            g.update(new)
