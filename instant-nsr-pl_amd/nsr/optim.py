"""AdamW over any number of tensors for a user's own training system (the reference's ``parse_optimizer`` builds
``torch.optim.AdamW``: systems/utils.py:314-325; the trainers of this package own their optimizers and do not need it)."""
import math
from collections import defaultdict

import numpy as np
import torch

from nsr_hip import NsrAdamwTensor, NsrError, check, device_guard, lib, ptr, stream_ptr
from nsr_hip.ops import DTYPE_CODES, timed

F32, F8 = torch.float32, torch.float8_e4m3fn
_DESCRIPTOR = np.dtype(NsrAdamwTensor)
# (of a list by map: the host side of a step of many tensors is these)
_address, _size, _contiguous = torch.Tensor.data_ptr, torch.Tensor.nbytes.__get__, torch.Tensor.is_contiguous
_dtype, _device = torch.Tensor.dtype.__get__, torch.Tensor.get_device
BLOCK = 256  # elements under one scale of the 8-bit moments (csrc/optim.hip); every tensor's moments start at a multiple of it


def _is_dense(t):
    """``t``'s elements fill one span of memory, in whatever order of its axes"""
    if t.is_contiguous():
        return True
    order = sorted(range(t.dim()), key=lambda d: (-t.stride(d), -t.shape[d]))
    return t.permute(order).is_contiguous()


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` (decoupled weight decay, bias correction) with all tensors updated in one launch per 64 of them (36
    with 8-bit moments, images or a learning rate on the device).

    ``state_bits=8``: moments in 8 bits with one float32 scale per 256 elements and moment (16.1 instead of 28 bytes of memory
    traffic per float32 parameter and step, 2.06 instead of 8 bytes of state).  They are rounded stochastically, with random bits
    made from (``rounding_seed``, step, element): the same run gives the same bits.  Tensors with fewer than ``min_8bit_size``
    elements keep 32-bit moments.

    ``max_grad_norm``: gradients are scaled by min(1, max_grad_norm / (norm + 1e-6)) with the norm over the gradients of all
    tensors; a step whose norm is not finite is left out whole.  ``grad_norm`` holds the last step's norm (a 0-dim GPU tensor that
    the next step overwrites).  Nothing is read back to the host.  ``max_grad_norm`` and ``capturable`` may be set later on; what a
    captured step does stays as captured.

    ``capturable=True``: the step count lives on the device and ``step`` may be captured into a graph; the learning rate that a
    replay uses is a group's ``lr`` tensor (0-dim or one element, float32, on the GPU) or, if it is a number, the captured one.

    ``modules``: ``tinycudann`` modules whose ``params`` are among the parameters: the fp16 image that their kernels read is
    written in the same pass (otherwise they cast ``params`` again in every forward pass).  ``refresh_images``: for parameters that
    were written from outside between replays of a captured forward pass.

    ``flat32`` / ``flat8``: the moments of all tensors as one buffer each (``state`` holds views of them); ``set_step`` and
    ``taken_steps``: the step count.

    Parameters are float32, float16 or bfloat16 (arithmetic and 32-bit moments in float32), dense and on one GPU; ``betas`` and
    ``eps`` are the same for all groups, ``lr`` and ``weight_decay`` are the group's.  Tensors whose ``grad`` is None are left
    as they are; the step count is one for all tensors.  An element whose gradient is not finite keeps its value and moments
    (8-bit ones are rounded again with their block, under its new scale).
    Works with ``torch.amp.GradScaler`` without a synchronisation of its own: gradients are unscaled in the pass, a step with a
    non-finite one is left out.  32-bit state dicts can be exchanged with ``torch.optim.AdamW``'s (which rounds the moments of
    16-bit parameters to their type)."""

    _step_supports_amp_scaling = True

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, *, state_bits=32, min_8bit_size=4096,
                 max_grad_norm=None, capturable=False, modules=(), rounding_seed=0):
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits is 8 or 32, got {state_bits}")
        max_grad_norm = self._checked_norm(max_grad_norm)
        if not 0 <= int(rounding_seed) < 1 << 32:
            raise ValueError(f"AdamW: rounding_seed is a 32-bit number, got {rounding_seed}")
        self._built = False
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))
        self._state_bits, self._min_8bit_size, self.rounding_seed = int(state_bits), int(min_8bit_size), int(rounding_seed)
        self._capturable, self._max_grad_norm = bool(capturable), None
        self._step, self._step_dev, self._hyper, self._partials = 0, None, None, None
        self._lay_out()
        self._images = self._image_modules(modules)
        self._shared_hyperparameters()
        for g in self.param_groups:
            self._learning_rate(g)
        self.capturable, self.max_grad_norm = capturable, max_grad_norm
        self._built = True

    # ---- settings ------------------------------------------------------------------------------------------------------------
    state_bits = property(lambda self: self._state_bits, doc="fixed at construction: the moments are laid out for it")
    min_8bit_size = property(lambda self: self._min_8bit_size, doc="fixed at construction: the moments are laid out for it")

    @property
    def capturable(self):
        return self._capturable

    @capturable.setter
    def capturable(self, value):
        if value:
            self._device_step()
        self._capturable = bool(value)

    @staticmethod
    def _checked_norm(value):
        if value is not None and not 0.0 < float(value) < math.inf:
            raise ValueError(f"AdamW: max_grad_norm {value}")
        return None if value is None else float(value)

    @property
    def max_grad_norm(self):
        return self._max_grad_norm

    @max_grad_norm.setter
    def max_grad_norm(self, value):
        value = self._checked_norm(value)
        if value is not None:
            self._device_step()
            if self._partials is None:
                room = lib.nsr_grad_squares_capacity(self._desc, len(self._ps))
                self._partials = torch.empty(room, dtype=torch.float64, device=self.device)
        self._max_grad_norm = value

    # ---- construction --------------------------------------------------------------------------------------------------------
    def _lay_out(self):
        """every tensor's place in the flat moments, its descriptor, and ``self.state`` as views of them"""
        items = [(p, i) for i, g in enumerate(self.param_groups) for p in g["params"]]
        spans = []
        for p, _ in items:
            if not p.is_cuda:
                raise NsrError("AdamW: parameters live on the GPU (there is no CPU path in the product library)")
            if p.dtype not in DTYPE_CODES:
                raise NsrError(f"AdamW: float32/float16/bfloat16 parameters, got {p.dtype}")
            if p.device != items[0][0].device:
                raise NsrError(f"AdamW: parameters on {p.device} and {items[0][0].device}")
            if not _is_dense(p):
                raise NsrError(f"AdamW: a parameter of shape {tuple(p.shape)} with strides {p.stride()} is not dense")
            if p.numel():
                spans.append((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()))
        spans.sort()
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("AdamW: two parameters share memory")
        self.device = items[0][0].device
        self._ps = [p for p, _ in items]
        self._group_of = [i for _, i in items]
        self._all_contiguous = all(p.is_contiguous() for p in self._ps)
        self._addresses = [p.data_ptr() for p in self._ps]
        self._kinds = [list(map(of, self._ps)) for of in (_size, _dtype, _device)]
        self._bits = [8 if self._state_bits == 8 and p.numel() >= self._min_8bit_size else 32 for p in self._ps]
        n = np.array([p.numel() for p in self._ps], dtype=np.int64)
        eight = np.array([b == 8 for b in self._bits])
        room = -(-n // BLOCK) * BLOCK
        # flat moments: tensor i has [at, at + numel) of the set of its width, zeros behind it up to the next multiple of BLOCK
        at = np.where(eight, np.cumsum(room * eight) - room, np.cumsum(room * ~eight) - room)
        self._at, total8, total32 = at.tolist(), int((room * eight).sum()), int((room * ~eight).sum())
        zeros = lambda n, dtype: torch.zeros(n, dtype=torch.uint8 if dtype is F8 else dtype, device=self.device).view(dtype)  # noqa: E731
        self.flat32 = {k: zeros(total32, F32) for k in ("exp_avg", "exp_avg_sq")} if total32 else {}
        self.flat8 = {}
        if total8:
            self.flat8 = {k: zeros(total8, F8) for k in ("exp_avg", "exp_avg_rms")}
            self.flat8["scales"] = torch.zeros(2, total8 // BLOCK, dtype=F32, device=self.device)
        self._desc = (NsrAdamwTensor * len(self._ps))()
        f = self._fields = np.frombuffer(self._desc, dtype=_DESCRIPTOR)
        f["n"], f["index0"], f["state_bits"] = n, at, self._bits
        f["params"] = self._addresses
        f["dtype"] = [DTYPE_CODES[p.dtype] for p in self._ps]
        for flat, size, which in ((self.flat32, 4, ~eight & (n > 0)), (self.flat8, 1, eight)):
            if flat and which.any():
                first, second = list(flat)[:2]
                f["exp_avg"][which] = flat[first].data_ptr() + size * at[which]
                f["exp_avg_sq"][which] = flat[second].data_ptr() + size * at[which]
        if total8:
            f["scales_m"][eight] = self.flat8["scales"].data_ptr() + 4 * (at[eight] // BLOCK)
            f["scales_r"][eight] = f["scales_m"][eight] + 4 * (total8 // BLOCK)
        self._bind_state()

    def _bind_state(self):
        """``self.state`` as views of the flat moments, in the parameters' shapes and orders of elements"""
        for flat, width in ((self.flat32, 32), (self.flat8, 8)):
            ps = [p for p, bits in zip(self._ps, self._bits) if bits == width and p.numel()]
            if not ps:
                continue
            room = [-(-p.numel() // BLOCK) * BLOCK for p in ps]
            views = {k: t.split(room) if k != "scales" else t.split([r // BLOCK for r in room], dim=1) for k, t in flat.items()}
            for i, p in enumerate(ps):
                s = self.state[p] = {}
                for k, v in views.items():
                    if k == "scales":
                        s[k] = v[i]
                    elif p.dim() == 1 and p.numel() == room[i]:
                        s[k] = v[i]
                    else:
                        s[k] = v[i].as_strided(p.shape, p.stride())

    def _image_modules(self, modules):
        place = {id(p): i for i, p in enumerate(self._ps)}
        found, images = [], {}  # (modules of one parameter share its image)
        for m in modules:
            if m.params.numel() == 0:
                continue
            i = place.get(id(m.params))
            if i is None or m.params.dtype != F32:
                raise ValueError("AdamW: `modules` are tinycudann modules whose float32 `params` are among the parameters")
            if i not in images:
                images[i] = torch.empty_like(m.params, dtype=torch.float16)
                self._desc[i].image = images[i].data_ptr()
            found.append((m, i, images[i]))
        return found

    def _image_owner(self, module, i):
        if module.params is not self._ps[i]:
            raise NsrError("AdamW: a module of `modules` has another `params` than at construction")
        return module.params

    def add_param_group(self, param_group):
        if getattr(self, "_built", False):
            raise NotImplementedError("AdamW: the parameters are fixed at construction (their moments lie in flat buffers)")
        super().add_param_group(param_group)

    def __getstate__(self):
        raise NotImplementedError("AdamW: copy an optimizer through state_dict() / load_state_dict()")

    # ---- hyperparameters -----------------------------------------------------------------------------------------------------
    def _shared_hyperparameters(self):
        g0 = self.param_groups[0]
        (b1, b2), eps = g0["betas"], g0["eps"]
        for g in self.param_groups:
            if tuple(g["betas"]) != (b1, b2) or g["eps"] != eps:
                raise NotImplementedError("AdamW: betas and eps are the same for all groups")
            if g.get("amsgrad") or g.get("maximize"):  # (a state dict of torch.optim.AdamW's)
                raise NotImplementedError("AdamW: neither amsgrad nor maximize")
            if not g["weight_decay"] >= 0.0:
                raise ValueError(f"AdamW: weight_decay {g['weight_decay']}")
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and eps >= 0.0):
            raise ValueError(f"AdamW: betas {(b1, b2)}, eps {eps}")
        return b1, b2, eps

    def _learning_rate(self, group):
        """(number, device pointer) of a group's learning rate"""
        lr = group["lr"]
        if isinstance(lr, torch.Tensor):
            if lr.numel() != 1 or lr.dtype != F32:
                raise ValueError(f"AdamW: a learning rate tensor has one float32 element, got {tuple(lr.shape)} {lr.dtype}")
            if self._capturable:
                if lr.device != self.device:
                    raise ValueError(f"AdamW: the learning rate of a capturable optimizer is on {self.device}, got {lr.device}")
                return 0.0, lr.data_ptr()
            lr = float(lr)
        if not lr >= 0.0:
            raise ValueError(f"AdamW: lr {lr}")
        return float(lr), None

    # ---- step count ----------------------------------------------------------------------------------------------------------
    def _device_step(self):
        if self._step_dev is None:
            self._step_dev = torch.full((1,), self._step, dtype=torch.int32, device=self.device)
            self._hyper = torch.zeros(8, dtype=F32, device=self.device)
        return self._step_dev, self._hyper

    def taken_steps(self):
        """optimizer steps taken, those left out not among them (synchronises where the count lives on the device)"""
        return self._step if self._step_dev is None else int(self._step_dev.item())

    def set_step(self, count):
        """the next step is number ``count`` + 1 (``count`` >= 0)"""
        if not 0 <= int(count) < (1 << 31) - 1:
            raise ValueError(f"AdamW: a step count of {count}")
        self._step = int(count)
        if self._step_dev is not None:
            self._step_dev.fill_(self._step)

    @property
    def grad_norm(self):
        """norm of the last step's gradients before clipping (None without ``max_grad_norm``)"""
        return self._hyper[5] if self._max_grad_norm is not None else None

    # ---- one step ------------------------------------------------------------------------------------------------------------
    def _gather(self):
        """this step's addresses in the descriptors; (host array, count, live parameters, tensors to keep until the launch)"""
        f, ps = self._fields, self._ps
        grads = [p.grad for p in ps]
        addresses = list(map(_address, ps))
        if addresses != self._addresses:
            self._check_moved()
            self._addresses = addresses
            f["params"] = addresses
        keep = []
        try:
            whole = self._all_contiguous and all(map(_contiguous, grads))
        except TypeError:  # (a gradient is None)
            whole = False
        if not whole:
            live = [i for i, g in enumerate(grads) if g is not None]
            for i in live:
                if grads[i].layout is not torch.strided:
                    raise NsrError(f"AdamW: a gradient of layout {grads[i].layout} is not supported")
            self._check_kinds([grads[i] for i in live], [[kind[i] for i in live] for kind in self._kinds])
            for i in live:
                p, g = ps[i], grads[i]
                if g.stride() != p.stride() and p.numel():  # in the parameter's order of elements
                    grads[i] = torch.empty_strided(p.shape, p.stride(), dtype=p.dtype, device=p.device)
                    with torch.no_grad():
                        grads[i].copy_(g)
            keep = grads
            if len(live) < len(ps):
                for i in live:
                    f["grad"][i] = grads[i].data_ptr()
                some = f[live]  # (a copy)
                return some.ctypes.data, len(live), [ps[i] for i in live], (keep, some)
        else:
            self._check_kinds(grads, self._kinds)
        f["grad"] = list(map(_address, grads))
        return self._desc, len(ps), ps, keep

    @staticmethod
    def _check_kinds(grads, kinds):
        # the kernel reads a gradient by its address with the parameter's type.  torch sees to it for ``p.grad = g``, but not for
        # ``p.grad.data = g`` or a ``grad_dtype`` of its own
        sizes, dtypes, devices = kinds
        if list(map(_size, grads)) != sizes or list(map(_dtype, grads)) != dtypes or list(map(_device, grads)) != devices:
            raise NsrError("AdamW: a gradient has another size, type or device than its parameter")

    def _check_moved(self):
        """parameters whose memory was replaced (``p.data = ...``) still have the layout that the moments were made for"""
        for i, p in enumerate(self._ps):
            if p.numel() != self._fields["n"][i] or DTYPE_CODES.get(p.dtype) != self._fields["dtype"][i] or \
                    p.device != self.device or not _is_dense(p) or (p.numel() and p.stride() != self._stride(i)):
                raise NsrError(f"AdamW: parameter {i} changed its shape, type, strides or device since construction")

    def _stride(self, i):
        return next(iter(self.state[self._ps[i]].values())).stride()

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        b1, b2, eps = self._shared_hyperparameters()
        capturing = torch.cuda.is_current_stream_capturing()
        if capturing and not self._capturable:
            raise NsrError("AdamW: only an optimizer with capturable=True can step inside a graph capture")
        scale, found = getattr(self, "grad_scale", None), getattr(self, "found_inf", None)
        if self._step_dev is None and (scale is not None or found is not None):
            self._device_step()  # (a step may be left out: only the device knows the count)
        f = self._fields
        rates = [self._learning_rate(g) for g in self.param_groups]
        if len(rates) == 1:
            f["lr"], f["lr_dev"] = rates[0][0], rates[0][1] or 0
            f["weight_decay"] = self.param_groups[0]["weight_decay"]
        else:
            f["lr"] = [rates[i][0] for i in self._group_of]
            f["lr_dev"] = [rates[i][1] or 0 for i in self._group_of]
            f["weight_decay"] = [self.param_groups[i]["weight_decay"] for i in self._group_of]
        desc, n, live, keep = self._gather()
        if n == 0:
            return loss
        with device_guard(self.device), timed("adamw_step", n):
            for m, i, image in self._images:
                p = self._image_owner(m, i)
                if m._shadow is not image or not m._shadow_trusted or m._shadow_key != (p.data_ptr(), p._version, p.device):
                    image.copy_(p.detach())  # first step, or the parameters were written from outside
            s = stream_ptr()
            if self._step_dev is None:
                self._step += 1
                step, hyper = self._step, None
            else:
                self._begin(desc, n, b1, b2, scale, found, s)
                step, hyper = 0, ptr(self._hyper)
            check(lib.nsr_adamw_tensors(desc, n, b1, b2, eps, step, hyper, 1.0, self.rounding_seed, s), "nsr_adamw_tensors")
        torch.autograd.graph.increment_version(live)
        for m, i, image in self._images:
            m.adopt_shadow(image)
            m._replayed = m._replayed or capturing
        return loss

    def refresh_images(self):
        """writes the ``modules``' fp16 images from their parameters.  An eager forward pass sees by itself that parameters were
        written from outside; a captured one reads the image that the last step left, so call this between such a write and the next
        replay (or take one eager step)"""
        with torch.no_grad():
            for m, i, image in self._images:
                image.copy_(self._image_owner(m, i))
                m.adopt_shadow(image)

    def _begin(self, desc, n, b1, b2, scale, found, stream):
        for t in (scale, found):
            if t is not None and (t.dtype != F32 or t.device != self.device or t.numel() != 1):
                raise NsrError("AdamW: grad_scale and found_inf are one float32 element on the parameters' device")
        step, hyper = self._step_dev.data_ptr(), self._hyper.data_ptr()
        scale = None if scale is None else scale.data_ptr()
        found = None if found is None else found.data_ptr()
        if self._max_grad_norm is None:
            check(lib.nsr_adamw_begin(step, hyper, b1, b2, None, 0, 0.0, scale, found, stream), "nsr_adamw_begin")
            return
        check(lib.nsr_adamw_begin_clipped(desc, n, self._partials.data_ptr(), self._partials.numel(), step, hyper, b1, b2,
                                          self._max_grad_norm, scale, found, stream), "nsr_adamw_begin_clipped")

    # ---- checkpoints ---------------------------------------------------------------------------------------------------------
    def state_dict(self):
        """torch's layout; every tensor's state holds the common ``step`` as well"""
        held, step = self.state, float(self.taken_steps())
        self.state = defaultdict(dict, {p: {"step": torch.tensor(step), **s} for p, s in held.items()})
        try:
            return super().state_dict()  # (its hooks see the whole)
        finally:
            self.state = held

    def load_state_dict(self, state_dict):
        """state of an optimizer with the same tensors and the same ``state_bits`` for each of them.  32-bit moments stay float32,
        also of 16-bit parameters, and take in those of 16 bits that ``torch.optim.AdamW`` keeps for them"""
        before, after = self._optimizer_load_state_dict_pre_hooks, self._optimizer_load_state_dict_post_hooks
        state_dict = state_dict.copy()
        for hook in before.values():
            state_dict = hook(self, state_dict) or state_dict
        self._load(state_dict)
        for hook in after.values():
            hook(self)

    def _load(self, state_dict):
        saved, steps = state_dict["state"], set()
        if any(g.get("amsgrad") or g.get("maximize") for g in state_dict["param_groups"]):
            raise NotImplementedError("AdamW: neither amsgrad nor maximize")
        for i, p in enumerate(self._ps):
            if i not in saved or not p.numel():
                continue
            for k, t in self.state[p].items():
                v = saved[i].get(k)
                if v is None or v.dtype not in ((F32, torch.float16, torch.bfloat16) if t.dtype is F32 else (t.dtype,)) or \
                        v.shape != t.shape:
                    raise ValueError(f"AdamW.load_state_dict: tensor {i} needs {k} {tuple(t.shape)} {t.dtype}, the state has "
                                     f"{None if v is None else (tuple(v.shape), v.dtype)}")
            if "step" not in saved[i]:
                raise ValueError(f"AdamW.load_state_dict: the state of tensor {i} has no step count")
            steps.add(float(saved[i]["step"]))
        if len(steps) > 1:
            raise ValueError(f"AdamW.load_state_dict: the tensors' step counts differ: {sorted(steps)}")
        rates = [g["lr"] for g in self.param_groups]
        hooks = self._optimizer_load_state_dict_pre_hooks, self._optimizer_load_state_dict_post_hooks
        self._optimizer_load_state_dict_pre_hooks, self._optimizer_load_state_dict_post_hooks = {}, {}
        try:  # the groups alone: torch would cast the moments to the parameters' types
            super().load_state_dict({"state": {}, "param_groups": state_dict["param_groups"]})
        finally:
            self._optimizer_load_state_dict_pre_hooks, self._optimizer_load_state_dict_post_hooks = hooks
        for g, lr in zip(self.param_groups, rates):
            if isinstance(lr, torch.Tensor):  # (a captured step reads this tensor: it keeps its place)
                lr.fill_(float(g["lr"]))
                g["lr"] = lr
        self._bind_state()
        for i, p in enumerate(self._ps):
            for k, t in self.state.get(p, {}).items():
                if i not in saved:
                    (t.view(torch.uint8) if t.dtype is F8 else t).zero_()
                elif t.dtype is F8:
                    t.view(torch.uint8).copy_(saved[i][k].to(self.device).view(torch.uint8))
                else:
                    t.copy_(saved[i][k])
        self.set_step(int(steps.pop()) if steps else 0)
